"""marlsoccer.optim (ms_adamw_step, ms_grad_clip) against a 64-bit AdamW, and what it refuses.

Bounds: with u = 2^-24, m = b1 m + c1 g rounds three times and its constants once each, so it is off by
at most 6 u (|b1 m| + |c1 g|); v likewise by 8 u v, its root by 5 u of itself. The update's factors
(the bias corrections, computed in float64 and rounded, the quotient, the products) add 8 roundings to
the 6 and 5, the clip factor 3 more with its own in g: 24 u of (|b1 m| + |c1 g|) lr / denominator, and
p itself rounds 3 times. A 16-bit parameter is rounded once more, to half a step. A moment of 8 bits is
off by half a step of e4m3: 2^-4 of its value among the normal ones, half of 2^-9 scales below 2^-6
scales (the scale itself is max / 448 within 2 u)."""
import math

import pytest

torch = pytest.importorskip("torch")

from marlsoccer import optim  # noqa: E402

gpu = pytest.mark.gpu
U = 2.0 ** -24


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


SHAPES = [(1,), (3,), (64, 66), (512,), (7, 5), (255,), (256,), (257,), (1000, 13), (0,), (4099,), (1, 3)]


def make(shapes, dtype, seed, device="cuda"):
    g = torch.Generator()
    g.manual_seed(seed)
    ps = [torch.randn(s, generator=g).mul_(0.1).to(dtype).to(device) for s in shapes]
    gs = [(torch.randn(s, generator=g) * math.exp(torch.randn((), generator=g).item())).to(dtype).to(device) for s in shapes]
    return ps, gs


class Exact:
    """AdamW in 64 bits; with 8 bits the caller puts the held moments back after every step."""

    def __init__(self, ps, lr, betas, eps, decay, clip):
        self.p = [p.double().cpu() for p in ps]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.t = [0] * len(self.p)
        self.hp = lr, betas, eps, decay, clip

    def step(self, gs):
        lr, (b1, b2), eps, decay, clip = self.hp
        gs = [None if g is None else g.double().cpu() for g in gs]
        self.norm = math.sqrt(sum(float(g.square().sum()) for g in gs if g is not None))
        c = min(1.0, clip / (self.norm + 1e-6)) if clip else 1.0
        self.size, self.msize = [0.0] * len(gs), [0.0] * len(gs)
        for i, g in enumerate(gs):
            if g is None:
                continue
            self.t[i] += 1
            t, g = self.t[i], g * c
            self.msize[i] = b1 * self.m[i].abs() + (1 - b1) * g.abs()
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            den = torch.sqrt(self.v[i] / (1 - b2 ** t)) + eps
            f = lr / (1 - b1 ** t)
            self.size[i] = f * self.msize[i] / den
            self.p[i] = self.p[i] * (1 - lr * decay) - f * self.m[i] / den


def within(name, got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{name}: worst excess {float((off - bound).max()):.3g}"


def check(ref, ps, moments, dtype, bits):
    eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tiny = 2.0 ** -126
    for i, p in enumerate(ps):
        raw = 24 * U * ref.size[i] + 3 * U * ref.p[i].abs() + tiny
        sub = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step among float16's subnormals
        within(f"p{i}", p, ref.p[i], raw + eps * (ref.p[i].abs() + raw) + sub)
        m, v = moments(i)
        if bits == 32:
            within(f"m{i}", m, ref.m[i], 9 * U * ref.msize[i] + tiny)
            within(f"v{i}", v, ref.v[i], 12 * U * ref.v[i] + tiny)
        elif p.numel():
            for name, got, want, err in (("m", m, ref.m[i], 9 * U * ref.msize[i]), ("r", v, ref.v[i].sqrt(), 8 * U * ref.v[i].sqrt())):
                n = want.numel()
                top = torch.nn.functional.pad(want.abs().reshape(-1), (0, -n % optim.BLOCK)).view(-1, optim.BLOCK).amax(1)
                scale = (top / 448).repeat_interleave(optim.BLOCK)[:n].view(want.shape)
                err = torch.as_tensor(err) + 4 * U * top.repeat_interleave(optim.BLOCK)[:n].view(want.shape)
                within(f"{name}{i}", got, want, (want.abs() + err) * 2.0 ** -4 + scale * 2.0 ** -10 * (1 + 8 * U) + err + 2.0 ** -99)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.5, 1e9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_steps_match_64_bits(dtype, clip, bits):
    need_gpu()
    lr, betas, eps, decay = 3e-3, (0.9, 0.99), 1e-5, 0.05
    ps, _ = make(SHAPES, dtype, 1)
    opt = optim.AdamW([torch.nn.Parameter(p) for p in ps], lr=lr, betas=betas, eps=eps, weight_decay=decay, max_grad_norm=clip, state_bits=bits)
    params = opt.param_groups[0]["params"]
    ref = Exact(ps, lr, betas, eps, decay, clip)
    for step in range(5):
        _, gs = make(SHAPES, dtype, 10 + step)
        ref.p = [p.detach().double().cpu() for p in params]  # each step is held to its own bound
        if step:
            held = [moments(i) for i in range(len(ps))]
            ref.m = [m.double().cpu() for m, _ in held]
            ref.v = [(v.double() ** (2 if bits == 8 else 1)).cpu() for _, v in held]
        for p, g in zip(params, gs):
            p.grad = g.clone()
        opt.step()
        ref.step(gs)

        def moments(i):
            s = opt.state[params[i]]
            if bits == 32:
                return s["exp_avg"], s["exp_avg_sq"]
            return (optim.moment_values(s["exp_avg"], s["exp_avg_scale"]), optim.moment_values(s["exp_avg_sq"], s["exp_avg_sq_scale"]))

        check(ref, [p.detach() for p in params], moments, dtype, bits)
        assert all(int(opt.state[p]["step"]) == step + 1 for p in params)
        assert all(torch.equal(p.grad, g) for p, g in zip(params, gs))
        if clip:
            assert abs(float(opt.last_grad_norm) - ref.norm) <= 2 * U * ref.norm


@gpu
def test_many_tensors_over_several_launches():
    """More tensors than one launch takes, groups with their own settings, a parameter without a
    gradient, and one norm over all of them."""
    need_gpu()
    shapes = [(5 + i % 37, 1 + i % 11) for i in range(131)]
    ps, gs = make(shapes, torch.float32, 3)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    opt = optim.AdamW([dict(params=params[:100]), dict(params=params[100:], lr=1e-2, weight_decay=0.0)], lr=1e-3, weight_decay=0.1, max_grad_norm=2.0)
    a, b = Exact(ps[:100], 1e-3, (0.9, 0.999), 1e-8, 0.1, None), Exact(ps[100:], 1e-2, (0.9, 0.999), 1e-8, 0.0, None)
    skip = 57
    norm = math.sqrt(sum(float(g.double().square().sum()) for i, g in enumerate(gs) if i != skip))
    scale = min(1.0, 2.0 / (norm + 1e-6))
    for p, g, i in zip(params, gs, range(131)):
        p.grad = None if i == skip else g
    opt.step()
    clipped = [None if i == skip else g.double() * scale for i, g in enumerate(gs)]
    a.step(clipped[:100])
    b.step(clipped[100:])
    assert abs(float(opt.last_grad_norm) - norm) <= 2 * U * norm
    for i, p in enumerate(params):
        if i == skip:
            assert torch.equal(p.detach(), ps[i]) and not opt.state[p]
            continue
        ref, j = (a, i) if i < 100 else (b, i - 100)
        within(f"p{i}", p.detach(), ref.p[j], 24 * U * ref.size[j] + 3 * U * ref.p[j].abs() + 2.0 ** -126)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_views_and_the_functional_form(bits):
    """Tensors cut out of one buffer at odd offsets; values around them stay as they were; the same
    bits as the aligned ones."""
    need_gpu()
    shapes = [(33,), (256,), (700,), (1025,)]
    ps, gs = make(shapes, torch.float32, 5)
    outs = []
    for off in (0, 1):
        lists = dict(p=[], g=[], m=[], v=[], s=[], ms=[], vs=[])
        pads = []
        for p, g in zip(ps, gs):
            for key, src, dt in (("p", p, torch.float32), ("g", g, torch.float32), ("m", torch.zeros_like(p), None), ("v", torch.zeros_like(p), None)):
                dt = dt or (optim.F8 if bits == 8 else torch.float32)
                buf = torch.full((p.numel() + 2 * off + 2,), 7.0, device="cuda").to(dt)
                buf[off:off + p.numel()] = src.to(dt)
                lists[key].append(buf[off:off + p.numel()])
                pads.append((buf, off, p.numel()))
            lists["s"].append(torch.zeros(1, dtype=torch.int64, device="cuda"))
            for key in ("ms", "vs"):
                lists[key].append(torch.zeros(optim.scales_for(p.numel()), device="cuda"))
        for _ in range(3):
            optim.adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lists["s"], lr=1e-2, max_grad_norm=1.0,
                             exp_avg_scales=lists["ms"] if bits == 8 else None, exp_avg_sq_scales=lists["vs"] if bits == 8 else None)
        for buf, o, n in pads:
            assert bool((buf[:o].float() == 7.0).all()) and bool((buf[o + n:].float() == 7.0).all())
        outs.append([t.float() for k in ("p", "m", "v", "ms", "vs") for t in lists[k]])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@gpu
def test_non_finite_gradients_pass_into_the_update():
    """As clip_grad_norm_ and AdamW have it: an infinite norm makes the factor 0 (0 times the infinite
    gradient is no number, the others' 0), a NaN reaches every parameter."""
    need_gpu()
    for bad, others_nan in ((float("inf"), False), (float("nan"), True)):
        ps, gs = make([(300,), (10,)], torch.float32, 6)
        params = [torch.nn.Parameter(p.clone()) for p in ps]
        opt = optim.AdamW(params, max_grad_norm=1.0, weight_decay=0.0)
        gs[0][7] = bad
        for p, g in zip(params, gs):
            p.grad = g
        opt.step()
        got = torch.isnan(params[0].detach()).cpu()
        assert got[7] and bool(got.all()) == others_nan and bool(torch.isnan(params[1]).all()) == others_nan
    # with 8 bits a NaN is held as one, and the rest of its block goes on
    ps, gs = make([(300,)], torch.float32, 7)
    p = torch.nn.Parameter(ps[0].clone())
    opt = optim.AdamW([p], state_bits=8)
    gs[0][7] = float("nan")
    p.grad = gs[0]
    opt.step()
    held = optim.moment_values(opt.state[p]["exp_avg"], opt.state[p]["exp_avg_scale"])
    assert int(torch.isnan(held).sum()) == 1 and int(torch.isnan(p.detach()).sum()) == 1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    need_gpu()
    ps, _ = make([(40, 9), (17,)], torch.bfloat16, 8)
    runs = []
    for reload in (False, True):
        params = [torch.nn.Parameter(p.clone()) for p in ps]
        opt = optim.AdamW(params, lr=1e-2, max_grad_norm=1.0, state_bits=bits)
        for step in range(4):
            _, gs = make([(40, 9), (17,)], torch.bfloat16, 20 + step)
            for p, g in zip(params, gs):
                p.grad = g
            if reload and step == 2:
                saved = opt.state_dict()
                opt = optim.AdamW(params, lr=1e-2, max_grad_norm=1.0, state_bits=bits)
                opt.load_state_dict(saved)
            opt.step()
        runs.append([p.detach().clone() for p in params] + [opt.state[p]["exp_avg"].float() for p in params])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_replays(bits):
    """A step in a graph counts its steps and reads the learning rate and the gradients anew; eager
    steps may come between."""
    need_gpu()
    shapes = [(66, 64), (64,), (3,)]
    ps, gs = make(shapes, torch.float32, 9)
    runs = []
    for graph in (False, True):
        params = [torch.nn.Parameter(p.clone()) for p in ps]
        lr = torch.full((), 1e-2, device="cuda")
        opt = optim.AdamW(params, lr=lr, max_grad_norm=0.5, state_bits=bits)
        for p, g in zip(params, gs):
            p.grad = g.clone()
        opt.step()
        if graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                opt.step()
        for k in range(5):
            lr.mul_(0.8)
            for p in params:
                p.grad.mul_(-0.9)
            if graph and k != 2:
                g.replay()
            else:
                opt.step()
            torch.cuda.synchronize()
        assert all(int(opt.state[p]["step"]) == 6 for p in params)
        runs.append([p.detach().clone() for p in params] + [opt.state[p]["exp_avg_sq"].float() for p in params])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@gpu
def test_agrees_with_torch_adamw():
    need_gpu()
    ps, _ = make([(64, 66), (64,)], torch.float32, 30)
    a, b = [[torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2)]
    mine, theirs = optim.AdamW(a, lr=1e-3, weight_decay=0.02, max_grad_norm=0.5), torch.optim.AdamW(b, lr=1e-3, weight_decay=0.02)
    for k in range(20):
        _, gs = make([(64, 66), (64,)], torch.float32, 40 + k)
        for p, q, g in zip(a, b, gs):
            p.grad, q.grad = g.clone(), g.clone()
        mine.step()
        torch.nn.utils.clip_grad_norm_(b, 0.5)
        theirs.step()
    for p, q in zip(a, b):  # each of 20 steps moves a parameter by about lr, each within 24 u and some for theirs
        assert float((p - q).abs().max()) <= 20 * (48 * U * 10 * 1e-3 + 6 * U)


# ---------------------------------------------------------------- refusals (CPU)

def test_refusals():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(max_grad_norm=0.0),
               dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="HIP device"):
        optim.AdamW([p]).step()
    z = lambda n=4, dt=torch.float32: torch.zeros(n, dtype=dt)  # noqa: E731
    good = dict(params=[z()], grads=[z()], exp_avg=[z()], exp_avg_sq=[z()], steps=[z(1, torch.int64)], lr=1e-3)

    def refuses(match, **kw):
        with pytest.raises(ValueError, match=match):
            optim.adamw_step(**{**good, **kw})

    refuses("HIP device")
    refuses("one for every parameter", grads=[])
    refuses("float32, bfloat16 or float16", params=[z(4, torch.float64)])
    refuses("of its parameter's type", grads=[z(4, torch.float16)])
    refuses("of its parameter's type", grads=[z(5)])
    refuses("contiguous", params=[torch.zeros(2, 8)[:, ::2]], grads=[torch.zeros(2, 4)])
    refuses("a moment", exp_avg=[z(3)])
    refuses("a moment", exp_avg_sq=[z(4, torch.float16)])
    refuses("one int64", steps=[z(1)])
    refuses("both given", exp_avg_scales=[z(1)])
    refuses("a moment", exp_avg_scales=[z(1)], exp_avg_sq_scales=[z(1)])
    f8 = dict(exp_avg=[z(4, optim.F8)], exp_avg_sq=[z(4, optim.F8)])
    refuses("scales", **f8, exp_avg_scales=[z(2)], exp_avg_sq_scales=[z(1)])
    refuses("positive", max_grad_norm=-1.0)
    refuses("workspace", workspace=z(7))
    refuses("grad_norm", grad_norm=z(2))
    refuses("lr must be", lr=z(2))


def test_a_tensor_given_twice_is_refused():
    """Two blocks would race on it (a shared count would rise once for all of a launch's tensors)."""
    def two(dt=torch.float32, n=4):
        return [torch.zeros(n, dtype=dt), torch.zeros(n, dtype=dt)]

    good = dict(params=two(), grads=two(), exp_avg=two(), exp_avg_sq=two(), steps=two(torch.int64, 1), lr=1e-3)
    for name in ("params", "exp_avg", "exp_avg_sq", "steps"):
        with pytest.raises(ValueError, match="given twice"):
            optim.adamw_step(**{**good, name: [good[name][0]] * 2})
    with pytest.raises(ValueError, match="given twice"):
        optim.adamw_step(**{**good, "exp_avg": good["exp_avg_sq"]})
    with pytest.raises(ValueError, match="HIP device"):  # a gradient is only read, and empty tensors have no address
        optim.adamw_step(**{**good, "grads": [good["grads"][0]] * 2})
    with pytest.raises(ValueError, match="HIP device"):
        optim.adamw_step(two(n=0), two(n=0), two(n=0), two(n=0), two(torch.int64, 1), lr=1e-3)


def test_c_entries_refuse_bad_arguments():
    from marlsoccer import _native as N
    L = N.lib()
    rows = (N.MsOptimTensor * 1)(N.MsOptimTensor(numel=4))
    step = lambda rows, bits=32, lr=1e-3, b1=0.9, work=16: L.ms_adamw_step(rows, 1, bits, lr, None, b1, 0.99, 1e-8, 0.0, 0, work, None)  # noqa: E731
    assert step(rows) == N.MS_ERR_INVALID_ARGUMENT and b"gradient" in L.ms_optim_last_error()
    rows[0].grad = 16
    assert step(rows) == N.MS_ERR_INVALID_ARGUMENT and b"step count" in L.ms_optim_last_error()
    rows[0].step = 16
    assert step(rows) == N.MS_ERR_INVALID_ARGUMENT and b"param" in L.ms_optim_last_error()
    assert step(rows, work=None) == N.MS_ERR_INVALID_ARGUMENT and b"workspace" in L.ms_optim_last_error()
    assert step(rows, bits=4) == N.MS_ERR_INVALID_ARGUMENT
    assert step(rows, lr=float("nan")) == N.MS_ERR_INVALID_ARGUMENT
    assert step(rows, b1=1.0) == N.MS_ERR_INVALID_ARGUMENT
    assert L.ms_grad_clip(rows, 1, 0.0, None, 16, None) == N.MS_ERR_INVALID_ARGUMENT
    rows[0].dtype = 5
    assert L.ms_grad_clip(rows, 1, 1.0, None, 16, None) == N.MS_ERR_INVALID_ARGUMENT


@gpu
def test_copies_and_torchs_own_state():
    """A deep copy goes on like the original; torch.optim.AdamW's state_dict is taken over."""
    import copy
    need_gpu()
    ps, _ = make([(20, 5), (7,)], torch.float32, 50)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    theirs = torch.optim.AdamW(params, lr=1e-3, weight_decay=0.02)

    def grads(k):
        for p, g in zip(params, make([(20, 5), (7,)], torch.float32, 60 + k)[1]):
            p.grad = g

    for k in range(3):
        grads(k)
        theirs.step()
    mine = optim.AdamW(params, lr=1e-3, weight_decay=0.02)
    mine.load_state_dict(theirs.state_dict())
    assert all(int(mine.state[p]["step"]) == 3 for p in params)
    grads(3)
    before = [p.detach().clone() for p in params]
    mine.step()
    mine_after = [p.detach().clone() for p in params]
    for p, b in zip(params, before):
        p.data.copy_(b)
    theirs.step()
    for p, a in zip(params, mine_after):
        assert float((p.detach() - a).abs().max()) <= 48 * U * 10 * 1e-3 + 6 * U  # one step's worth of both's roundings
    twin = copy.deepcopy(mine)
    assert twin.state_bits == 32 and twin.max_grad_norm is None
    twin.step()  # its parameters have no gradients' history of their own, but deep copies of them


@gpu
def test_a_first_step_is_not_captured():
    need_gpu()
    ps, gs = make([(8, 3)], torch.float32, 70)
    p = torch.nn.Parameter(ps[0].clone())
    p.grad = gs[0]
    opt = optim.AdamW([p], max_grad_norm=1.0)
    torch.cuda.synchronize()
    count = torch.zeros(1, device="cuda")
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        count.add_(1)
        with pytest.raises(RuntimeError, match="before the capture"):
            opt.step()
    assert torch.equal(p.detach(), ps[0])
    opt.step()
    assert int(opt.state[p]["step"]) == 1


@gpu
def test_a_saved_parameter_that_was_stepped_refuses_its_backward():
    need_gpu()
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    opt = optim.AdamW([p])
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---------------------------------------------------------------- 8-bit moments over many steps

def eight_bit_lists(m, r, steps=None):
    """The lists of one tensor whose held moments are m and r (root of the second), as quantised to nearest."""
    def held(x):
        f = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % optim.BLOCK)).view(-1, optim.BLOCK)
        top = f.abs().amax(1)
        return (f * (448 / top)[:, None]).to(optim.F8).view(-1)[:x.numel()].view(x.shape).contiguous(), top / 448
    (mc, ms), (rc, rs) = held(m), held(r)
    return dict(exp_avg=[mc], exp_avg_sq=[rc], exp_avg_scales=[ms], exp_avg_sq_scales=[rs])


@gpu
def test_stochastic_rounding_keeps_the_expected_moments():
    """One step from the same state under many step counts: the moments are off by less than a step of their
    codes each time, and their mean over the counts is the unrounded value. A mean of K draws between two
    neighbours has a deviation of at most step / (2 sqrt(K)); 6 of them hold for 2 x 5,003 values with a
    probability of 1 - 10,006 x 2e-9. The odds have 16 bits, cut: a bias of at most 2^-16 steps, and
    float32's roundings of the moment before it (9 u and 8 u of its terms, the module's comment) and of the
    scaled value (2 u). A root below the smallest code is held as that code. The same count gives the same bits."""
    need_gpu()
    n, K, b1, b2 = 5003, 600, 0.9, 0.999
    g = torch.Generator().manual_seed(11)
    size = torch.exp(1.5 * torch.randn(n, generator=g))
    m0, r0, grad = (torch.randn(n, generator=g) * size).cuda(), (torch.rand(n, generator=g) * size).cuda(), (torch.randn(n, generator=g) * size).cuda()
    start = eight_bit_lists(m0, r0)
    held_m = optim.moment_values(start["exp_avg"][0], start["exp_avg_scales"][0]).double()
    held_r = optim.moment_values(start["exp_avg_sq"][0], start["exp_avg_sq_scales"][0]).double()
    terms = b1 * held_m.abs() + (1 - b1) * grad.double().abs()
    want = (b1 * held_m + (1 - b1) * grad.double(), (b2 * held_r.square() + (1 - b2) * grad.double().square()).sqrt())
    sums = [torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2)]
    for k in range(K):
        outs = []
        for again in range(2 if k == 0 else 1):
            count = torch.tensor([k], device="cuda")
            lists = {key: [t[0].clone()] for key, t in start.items()}
            optim.adamw_step([torch.zeros(n, device="cuda")], [grad], steps=[count], lr=1e-3, betas=(b1, b2), rounding="stochastic", **lists)
            outs.append([optim.moment_values(lists[c][0], lists[s][0]).double() for c, s in (("exp_avg", "exp_avg_scales"), ("exp_avg_sq", "exp_avg_sq_scales"))])
        assert all(torch.equal(a, b) for a, b in zip(outs[0], outs[-1]))
        for j, (got, s) in enumerate(zip(outs[0], ("exp_avg_scales", "exp_avg_sq_scales"))):
            scale = lists[s][0].double().repeat_interleave(optim.BLOCK)[:n]
            if j == 1 and k == 0:
                want = (want[0], torch.maximum(want[1], scale * 2.0 ** -9))
            unit = torch.exp2(torch.floor(torch.log2((want[j].abs() / scale).clamp(min=2.0 ** -6))) - 3) * scale  # a step of the codes there
            err = (9 * U * terms if j == 0 else 8 * U * want[1]) + 2 * U * want[j].abs()
            assert bool(((got - want[j]).abs() <= unit + err).all()), (k, j)
            sums[j] += got
            if k == K - 1:
                off = (sums[j] / K - want[j]).abs()
                bound = unit * (6 / (2 * math.sqrt(K)) + 2.0 ** -16) + err
                assert bool((off <= bound).all()), (j, float((off / bound).max()))


@gpu
@pytest.mark.parametrize("change", ["steady", "half of them grow four times", "half of them shrink to a tenth", "one was large for half the time"])
def test_stochastic_moments_follow_64_bits_over_thousands_of_steps(change):
    """Never brought back to the 64-bit moments. A root r moves by at most 0.0005 |g^2 / v - 1| of itself a step,
    0.001 on average, and so does the largest, whose scale shifts the codes; a rounding's variance is at most
    its step (2^-3 r) times the shift: 2.5e-4 r^2 a step, forgotten at 0.001 a step, so 0.125 r^2 in all; where
    gradients fall, v falls by 0.001 a step and what was off stays as it was against it: 1.25e-4 for up to
    3,000 steps and what was there, 0.5 r^2. The mean of the roots: v is too large by that variance on
    average, a root by half of it at most while steady (0.0625), and by a quarter where it is not
    stationary; the mean of 2,048 independent values is known to 0.016."""
    need_gpu()
    n, T, at, b2 = 2048, 4000, 1000, 0.999
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = optim.AdamW([p], lr=1e-6, betas=(0.9, b2), weight_decay=0.0, state_bits=8, rounding="stochastic")
    some = torch.arange(n, device="cuda") % 2 == 0
    one = torch.arange(n, device="cuda") % optim.BLOCK == 3
    v = torch.zeros(n, dtype=torch.float64, device="cuda")
    for t in range(T):
        g = torch.randn(n, generator=gen, device="cuda")
        if change == "half of them grow four times" and t >= at:
            g = torch.where(some, 4 * g, g)
        elif change == "half of them shrink to a tenth" and t >= at:
            g = torch.where(some, 0.1 * g, g)
        elif change == "one was large for half the time" and t < T // 2:
            g = torch.where(one, 30 * g, g)
        p.grad = g
        opt.step()
        v = b2 * v + (1 - b2) * g.double().square()
    s = opt.state[p]
    ratio = optim.moment_values(s["exp_avg_sq"], s["exp_avg_sq_scale"]).double() / v.sqrt()
    falls = change in ("half of them shrink to a tenth", "one was large for half the time")
    for part in (some & ~one, ~some & ~one):
        assert abs(float(ratio[part].mean()) - 1) <= (0.25 if falls else 0.0625 + 0.05), change
        assert float((ratio[part] - 1).square().mean()) <= (0.5 if falls else 0.125), change


@gpu
def test_stochastic_first_moment_reaches_a_constant_gradient():
    """m goes from 0 to g by a tenth of the distance a step; to nearest it stops where a tenth is half a step
    of the codes, far below g. The deviation of a rounding that keeps the expectation: at most half a step (2^-4
    of the value) each, forgotten by 0.9 a step: 2^-4 / sqrt(1 - 0.81) = 0.144 of the value, and the
    mean over 1,024 of them is known to 0.0045."""
    need_gpu()
    n = 1024
    g = torch.linspace(0.05, 1.0, n, device="cuda")[torch.randperm(n, generator=torch.Generator().manual_seed(3)).cuda()]
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = optim.AdamW([p], lr=1e-6, state_bits=8, rounding="stochastic")
    for _ in range(200):  # 0.9^200 = 7e-10 is left of the start
        p.grad = g
        opt.step()
    ratio = optim.moment_values(opt.state[p]["exp_avg"], opt.state[p]["exp_avg_scale"]) / g
    assert abs(float(ratio.mean()) - 1) <= 6 * 0.0045
    assert float((ratio - 1).square().mean()) <= 0.144 ** 2


def test_rounding_is_checked_and_named():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(state_bits=8, rounding="up"), dict(state_bits=32, rounding="stochastic"), dict(rounding="nearest")):
        with pytest.raises(ValueError, match="rounding"):
            optim.AdamW([p], **kw)
    with pytest.warns(UserWarning, match="stochastic"):
        optim.AdamW([p], state_bits=8)
    import copy
    import warnings
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        optim.AdamW([p])
        optim.AdamW([p], state_bits=8, rounding="nearest")
        assert copy.deepcopy(optim.AdamW([p], state_bits=8, rounding="stochastic")).rounding == "stochastic"
    one = dict(params=[torch.zeros(4)], grads=[torch.zeros(4)], exp_avg=[torch.zeros(4)], exp_avg_sq=[torch.zeros(4)], steps=[torch.zeros(1, dtype=torch.int64)], lr=1e-3)
    with pytest.raises(ValueError, match="rounding"):
        optim.adamw_step(**one, rounding="down")
    from marlsoccer import _native as N
    rows = (N.MsOptimTensor * 1)(N.MsOptimTensor(numel=4, grad=16, step=16, param=16, exp_avg=16, exp_avg_sq=16))
    for bits in (256, 32 | 256, 8 | 512):
        assert N.lib().ms_adamw_step(rows, 1, bits, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, 0, 16, None) == N.MS_ERR_INVALID_ARGUMENT


@gpu
@pytest.mark.parametrize("rounding", ["nearest", "stochastic"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), 1e25], ids=["inf", "minus inf", "nan", "a square past float32"])
def test_a_non_finite_moment_of_8_bits_stays_alone(bad, rounding):
    """Its own parameter is lost (as with 32 bits); the rest of its block goes on as without it. 1e25: only
    the second moment overflows, and the first is the block's largest, so there only the second is compared."""
    need_gpu()
    runs = []
    for value in (0.0, bad):
        (p,), _ = make([(700,)], torch.float32, 90)
        p = torch.nn.Parameter(p)
        opt = optim.AdamW([p], lr=1e-2, state_bits=8, rounding=rounding)
        for k in range(4):
            _, (g,) = make([(700,)], torch.float32, 91 + k)
            g[300] = value if k == 1 else 0.0
            p.grad = g
            opt.step()
            s = opt.state[p]
            if k == 1:
                m, r = (optim.moment_values(s[c], s[c + "_scale"]) for c in ("exp_avg", "exp_avg_sq"))
                m1, r1 = m.clone(), r.clone()
        runs.append((p.detach(), m1, r1))
    (p0, m0, r0), (p1, m1, r1) = runs
    others = torch.arange(700, device="cuda") != 300
    assert torch.isnan(p1[300]) and torch.isnan(r1[300]) and torch.equal(r0[others], r1[others])
    if not math.isfinite(bad):
        assert torch.isnan(m1[300]) and torch.equal(m0[others], m1[others]) and torch.equal(p0[others], p1[others])


def test_a_state_of_another_update_is_refused_when_loaded():
    """Saved by torch's optimizers with settings that this update does not have, or with moments of other
    bits; nothing of it is taken over."""
    def params():
        return [torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(3))]

    def saved(cls, **kw):
        ps = params()
        opt = cls(ps, **kw)
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
        return opt.state_dict()

    T = torch.optim
    mine = lambda bits=32: optim.AdamW(params(), lr=0.5, state_bits=bits, rounding="stochastic" if bits == 8 else None)  # noqa: E731
    for cls, kw, match in ((T.AdamW, dict(maximize=True), "maximize"), (T.AdamW, dict(amsgrad=True), "amsgrad"),
                           (T.Adam, dict(weight_decay=0.1), "decoupled")):
        opt = mine()
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(saved(cls, **kw))
        assert not opt.state and opt.param_groups[0]["lr"] == 0.5
    with pytest.raises(ValueError, match="maximize"):
        optim.AdamW([dict(params=params(), maximize=True)])
    with pytest.raises(TypeError, match="dict"):  # torch's own
        mine().add_param_group(params())
    with pytest.raises(ValueError, match="moments are"):
        mine(8).load_state_dict(saved(T.AdamW))
    eight = mine(8)
    for p in eight.param_groups[0]["params"]:
        eight._state_of(p)
    with pytest.raises(ValueError, match="moments are"):
        mine().load_state_dict(eight.state_dict())
    mine(8).load_state_dict(eight.state_dict())
    for cls, kw in ((T.AdamW, dict(weight_decay=0.1, lr=0.25)), (T.Adam, dict(lr=0.25))):
        opt = mine()
        opt.load_state_dict(saved(cls, **kw))
        assert opt.param_groups[0]["lr"] == 0.25 and all(int(s["step"]) == 1 for s in opt.state.values())


def test_scales_and_gradients_that_are_written_elsewhere_are_refused():
    """Waves of one launch would race on them: a scale array for both moments or for two tensors, and a
    gradient that is also another tensor's parameter or moment."""
    def two(dt=torch.float32, n=4):
        return [torch.zeros(n, dtype=dt), torch.zeros(n, dtype=dt)]

    good = dict(params=two(), grads=two(), exp_avg=two(optim.F8), exp_avg_sq=two(optim.F8), steps=two(torch.int64, 1), exp_avg_scales=two(n=1),
                exp_avg_sq_scales=two(n=1), lr=1e-3)
    for bad in (dict(exp_avg_scales=good["exp_avg_sq_scales"]), dict(exp_avg_scales=[good["exp_avg_scales"][0]] * 2),
                dict(exp_avg_sq_scales=[good["exp_avg_sq_scales"][1]] * 2), dict(grads=good["params"][::-1])):
        with pytest.raises(ValueError, match="given twice"):
            optim.adamw_step(**{**good, **bad})
    moments = two()
    with pytest.raises(ValueError, match="given twice"):
        optim.adamw_step(two(), moments, moments, two(), two(torch.int64, 1), lr=1e-3)
    with pytest.raises(ValueError, match="HIP device"):
        optim.adamw_step(**good)
    with pytest.raises(ValueError, match="HIP device"):  # empty tensors have no address
        none = [torch.zeros(0), torch.zeros(0)]
        optim.adamw_step(two(n=0), two(n=0), two(optim.F8, 0), two(optim.F8, 0), two(torch.int64, 1), lr=1e-3, exp_avg_scales=none, exp_avg_sq_scales=none)


def test_a_norm_that_nothing_computes_is_refused():
    one = dict(params=[torch.zeros(4)], grads=[torch.zeros(4)], exp_avg=[torch.zeros(4)], exp_avg_sq=[torch.zeros(4)], steps=[torch.zeros(1, dtype=torch.int64)], lr=1e-3)
    with pytest.raises(ValueError, match="no norm is computed"):
        optim.adamw_step(**one, grad_norm=torch.zeros(1))
    with pytest.raises(ValueError, match="HIP device"):
        optim.adamw_step(**one, grad_norm=torch.zeros(1), max_grad_norm=float("inf"))


@gpu
def test_an_infinite_max_grad_norm_gives_the_norm_and_clips_nothing():
    need_gpu()
    ps, gs = make([(300,), (7,)], torch.float32, 95)
    outs = []
    for kw in ({}, dict(max_grad_norm=float("inf"), grad_norm=torch.zeros((), device="cuda"))):
        lists = [[t.clone() for t in ps], gs, [torch.zeros_like(t) for t in ps], [torch.zeros_like(t) for t in ps], [torch.zeros(1, dtype=torch.int64, device="cuda") for _ in ps]]
        optim.adamw_step(*lists, lr=1e-2, **kw)
        outs.append(lists[0])
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and abs(float(kw["grad_norm"]) - norm) <= 2 * U * norm


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_deep_copy_steps_like_the_original(bits):
    """The copy's parameters come without gradients (a Parameter's deep copy has none): given the same ones,
    copy and original take the same steps, each with its own moments, counts and workspace."""
    import copy
    need_gpu()
    shapes = [(20, 5), (700,)]
    ps, _ = make(shapes, torch.float32, 97)
    mine = optim.AdamW([torch.nn.Parameter(p) for p in ps], lr=1e-2, max_grad_norm=0.5, state_bits=bits, rounding="stochastic" if bits == 8 else None)

    def step(opt, k):
        for p, g in zip(opt.param_groups[0]["params"], make(shapes, torch.float32, 98 + k)[1]):
            p.grad = g
        opt.step()

    def held(opt):
        return [t for p in opt.param_groups[0]["params"] for t in (p.detach(), *opt.state[p].values())]

    for k in range(2):
        step(mine, k)
    twin = copy.deepcopy(mine)
    assert {t.data_ptr() for t in held(mine)}.isdisjoint(t.data_ptr() for t in held(twin)) and not twin._work
    for k in (2, 3):
        step(mine, k)
        assert all(int(twin.state[p]["step"]) == k for p in twin.param_groups[0]["params"])  # not moved by the original's step
        step(twin, k)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(held(mine), held(twin)))
        assert torch.equal(mine.last_grad_norm, twin.last_grad_norm)
    assert {w.data_ptr() for w in mine._work[ps[0].device]}.isdisjoint(w.data_ptr() for w in twin._work[ps[0].device])


@gpu
def test_there_is_no_norm_before_a_clipped_step():
    need_gpu()
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    p.grad = torch.full_like(p, 3.0)
    opt = optim.AdamW([p])
    opt.step()
    assert opt.last_grad_norm is None
    opt.max_grad_norm = 1.0
    opt.step()
    assert float(opt.last_grad_norm) == 6.0


@gpu
@pytest.mark.parametrize("rounding", ["stochastic", "nearest"])
@pytest.mark.parametrize("small", [1e-5, 1e-6, 1e-7])
def test_values_far_below_their_blocks_largest_take_no_long_steps(small, rounding):
    """One value of 256 has gradients of size 1, the others of `small`, near or under the smallest code
    (4.4e-6 of the largest). Unrounded, |m| <= (1 - b1) / sqrt((1 - b2) (1 - b1^2 / b2)) r = 7.3 r by
    Cauchy and Schwarz: no step is longer than 7.3 lr. Rounded,
    m is up to a code higher and r as much lower, but not below one code: 4.4e-6 of the largest, whose
    own m / r is at most 7.3 too. So (7.3 small + 7.3 x 4.4e-6) over 4.4e-6 at most where r is one code, less
    above, and the bias corrections of the first 20 steps raise it by sqrt(1 - 0.999^t) / (1 - 0.9^t) < 1. To
    nearest a root of one code stays there until 0.999 + 0.001 g^2 passes 1.5^2: g, and so m, is below 36 of it."""
    need_gpu()
    n, lr = 1024, 1e-3
    gen = torch.Generator(device="cuda").manual_seed(7)
    size = torch.where(torch.arange(n, device="cuda") % optim.BLOCK == 5, 1.0, small)
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = optim.AdamW([p], lr=lr, eps=1e-8, weight_decay=0.0, state_bits=8, rounding=rounding)
    longest = torch.zeros((), device="cuda")
    for t in range(500):
        before = p.detach().clone()
        g = torch.randn(n, generator=gen, device="cuda") * size
        p.grad = g * (torch.rand(n, generator=gen, device="cuda") < 0.5)  # half of them without a gradient
        opt.step()
        longest = torch.maximum(longest, (p.detach() - before).abs().max())
    one = 2.0 ** -9 / 448
    assert float(longest) <= lr * (7.3 if rounding == "stochastic" else 36) * (1 + min(small, one) / one) * (1 + 2.0 ** -3)
