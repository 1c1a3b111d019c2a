"""Agents with a sequence memory: the rollout, its replay by the update, evaluation, and the whole
loop with the optimiser."""
import pytest

torch = pytest.importorskip("torch")

import sequence_reference as ref  # noqa: E402

from marlsoccer.memory import SequenceMemory  # noqa: E402
from marlsoccer.rollout import Agent, DeviceRollout, RunningMeanStd  # noqa: E402

gpu = pytest.mark.gpu


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def test_an_agent_without_memory_keeps_its_checkpoint_layout():
    assert not any(k.startswith("memory") for k in Agent().state_dict())
    keys = Agent(memory=SequenceMemory()).state_dict()
    assert {"memory.in_proj.weight", "memory.A_log", "memory.conv_weight"} <= set(keys)


def plain_memory(m, x, starts, state):
    """SequenceMemory.forward in 64 bits on the CPU."""
    d = lambda t: t.detach().double().cpu()  # noqa: E731
    xz = d(x) @ d(m.in_proj.weight).t()
    u, z = xz.chunk(2, -1)
    u, conv, _ = ref.conv(u, m.conv_weight, m.conv_bias, state[0], starts)
    r, B, C = (u @ d(m.x_proj.weight).t()).split((m.rank, m.states, m.states), -1)
    y, h, _ = ref.scan(u, r @ d(m.rate_proj.weight).t(), -torch.exp(d(m.A_log)), B, C, m.skip, z, m.rate_bias, state[1], starts)
    return d(x) + y @ d(m.out_proj.weight).t(), conv, h


@gpu
def test_steps_and_sequences_match_the_plain_form():
    """Both forms against 64 bits. The projections are products of at most 128 terms in float32 (an error
    of 128 u of their size) and feed the recurrences, whose outputs are held to 1e-4 here; each operator's
    own bound is tests/test_sequence.py's."""
    need_gpu()
    torch.manual_seed(0)
    T, R = 20, 6
    m = SequenceMemory(channels=96).cuda()
    x = torch.randn(T, R, 66).cuda()
    starts = torch.rand(T, R).cuda() < 0.1
    state = tuple(torch.randn_like(s) for s in m.init_state(R, "cuda"))
    want, conv, h = plain_memory(m, x, starts, state)
    y, (c1, h1) = m(x, starts, state)
    stepped = tuple(s.clone() for s in state)
    ys = torch.stack([m.step(x[t], stepped, starts[t]) for t in range(T)])
    for got, c, s in ((y, c1, h1), (ys, *stepped)):
        for a, b in ((got, want), (c, conv), (s, h)):
            assert float((a.detach().double().cpu() - b).abs().max()) <= 1e-4 * (1 + float(b.abs().max()))


def make(N, T, graph=False, config=None, **kw):
    from marlsoccer import SoccerBatch
    torch.manual_seed(0)
    agent = Agent(memory=SequenceMemory()).cuda()
    b = SoccerBatch(N, config=config)
    b.reset(seed=19)
    return agent, b, DeviceRollout(b, agent, RunningMeanStd((66,), device="cuda"), T, seed=5, graph=graph, update_normalizer=False, **kw)


def short_config(steps):
    from marlsoccer.config import load_config
    cfg = load_config()
    cfg["simulation"]["max_steps"] = steps
    return cfg


@gpu
def test_rollout_replays_as_one_sequence():
    """What the rollout's single steps stored is what the update computes from the stored sequences and
    the state before them, across episode ends."""
    need_gpu()
    N, T = 24, 30
    agent, b, ro = make(N, T, config=short_config(13))
    assert ro.policy == "torch"
    with pytest.raises(ValueError, match="memory"):
        DeviceRollout(b, agent, ro.normalizer, T, policy="fused")
    for _ in range(2):
        out = ro.collect()
        assert out["dones"].any()
        x = ro.normalizer.normalize(out["obs"].reshape(-1, 66)).view(T, 2 * N, 66)
        y, state = agent.memory(x, out["dones"].reshape(T, -1).bool(), out["memory_state"])
        value = agent.get_value(y.reshape(-1, 66)).view(T, N, 2)
        assert float((value - out["values"]).abs().max()) <= 1e-4  # float32 products in another order
        for a, c in zip(state, ro.memory_state):
            assert float((a - c).abs().max()) <= 1e-4 * (1 + float(c.abs().max()))
        plain = agent.get_value(x.reshape(-1, 66)).view(T, N, 2)
        assert float((plain - out["values"]).abs().max()) > 1e-3  # the memory does something
    b.close()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_graph_rollout_matches_eager(dtype):
    need_gpu()
    runs = []
    for graph in (False, True):
        agent, b, ro = make(32, 9, graph, short_config(7), policy_dtype=dtype)
        outs = []
        for _ in range(4):
            out = ro.collect()
            outs += [out[k].clone() for k in ("obs", "actions", "values", "dones", "rewards")] + [s.clone() for s in ro.memory_state + out["memory_state"]]
        runs.append(outs)
        b.close()
    for a, c in zip(*runs):
        assert torch.equal(a, c)


@gpu
def test_evaluate_with_memory():
    need_gpu()
    from marlsoccer.evaluate import evaluate
    torch.manual_seed(0)
    agent = Agent(memory=SequenceMemory()).cuda()
    rms = RunningMeanStd(device="cuda")
    a = evaluate(agent, rms, 8, seed=3, config=short_config(40))
    g = evaluate(agent, rms, 8, seed=3, config=short_config(40), graph=True)
    assert (a["returns"] == g["returns"]).all() and (a["score"] == g["score"]).all()
    agent.memory = None
    plain = evaluate(agent, rms, 8, seed=3, config=short_config(40))
    assert (a["returns"] != plain["returns"]).any()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_collect_update_loop(bits):
    """Rollout (a replayed graph from the third on), replay through the memory, gradients to every
    parameter, the optimiser's step in place: the graph goes on reading the parameters."""
    need_gpu()
    from marlsoccer.optim import AdamW
    N, T = 16, 12
    agent, b, ro = make(N, T, True, short_config(9))
    opt = AdamW(agent.parameters(), lr=2.5e-4, eps=1e-5, weight_decay=0.0, max_grad_norm=0.5, state_bits=bits)
    at = None
    for it in range(4):
        out = ro.collect()
        if it > 1:
            assert ro._graph is at  # not captured again
        at = ro._graph
        x = ro.normalizer.normalize(out["obs"].reshape(-1, 66)).view(T, 2 * N, 66)
        y, _ = agent.memory(x, out["dones"].reshape(T, -1).bool(), out["memory_state"])
        _, logprob, entropy, value = agent.get_action_and_value(y.reshape(-1, 66), out["actions"].reshape(-1, 3))
        ratio = (logprob - out["logprobs"].reshape(-1)).exp()
        assert float((ratio - 1).abs().max()) <= 1e-3
        loss = -(ratio * out["rewards"].reshape(-1)).mean() + (value.squeeze(-1) - 1.0).square().mean() - 0.01 * entropy.mean()
        loss.backward()
        before = [p.detach().clone() for p in agent.parameters()]
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in agent.parameters())
        assert all(bool(p.grad.any()) for n, p in agent.named_parameters() if n.startswith("memory"))
        opt.step()
        opt.zero_grad()
        assert all(bool(torch.isfinite(p).all()) for p in agent.parameters())
        assert any(not torch.equal(p, q) for p, q in zip(before, agent.parameters()))
    b.close()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_next_value_is_the_next_rollouts_first(graph, dtype):
    """The value for bootstrapping goes through the memory and leaves its state and the generator alone: the
    next rollout, with the same parameters and statistics, stores it first. The products may be summed in
    another order: 1e-4 in float32 as above, and in bfloat16 the five layers' roundings of a different
    order, 2^-8 each of values of the size of 1."""
    need_gpu()
    N, T = 24, 15
    agent, b, ro = make(N, T, graph, short_config(13), policy_dtype=dtype)
    for _ in range(3):
        ro.collect()
        before, draws = [s.clone() for s in ro.memory_state], ro.gen.get_state()
        value = ro.next_value()
        assert value.shape == (N, 2) and value.dtype == torch.float32
        assert all(torch.equal(a, c) for a, c in zip(before, ro.memory_state)) and torch.equal(draws, ro.gen.get_state())
        x = ro.normalizer.normalize(ro.next_obs.reshape(-1, 66))
        plain = agent.get_value(x).view(N, 2).detach()
        first = ro.collect()["values"][0]
        assert float((value - first).abs().max()) <= (1e-4 if dtype == torch.float32 else 5 * 2.0 ** -8)
        if dtype == torch.float32:
            # a value without the memory would fail the line above: all that is asked of it is to be further off than that allows
            assert float((plain - first).abs().max()) > 1e-4
    b.close()


@gpu
@pytest.mark.parametrize("policy", ["fused", "torch"])
def test_next_value_without_memory(policy):
    need_gpu()
    from marlsoccer import SoccerBatch
    torch.manual_seed(0)
    agent = Agent().cuda()
    b = SoccerBatch(16, config=short_config(13))
    b.reset(seed=3)
    ro = DeviceRollout(b, agent, RunningMeanStd((66,), device="cuda"), 8, seed=5, update_normalizer=False, policy=policy)
    ro.collect()
    value = ro.next_value()
    assert float((value - ro.collect()["values"][0]).abs().max()) <= 1e-4
    b.close()


def test_a_state_of_another_type_is_taken_in_the_activations_type():
    """Without a device: the state's type is no longer what the call is refused for."""
    m = SequenceMemory()
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        with pytest.raises(ValueError, match="HIP device"):
            m(torch.zeros(3, 2, 66), None, m.init_state(2, dtype=dtype))


@gpu
@pytest.mark.parametrize("again", ["float32", "autocast"])
def test_bf16_rollout_replays(again):
    """A rollout under bfloat16 replayed by the update in float32, as documented, and under the same autocast.
    The critic under bfloat16 is within 2e-2 of float32 (tests/test_policy.py); the memory adds 128 products
    of roundings to 2^-8 (the projections' in and out, the activations between them), some four of them in a
    row, of a sum below 0.5: 8e-3 a feature, 0.064 over 66 of them at most, through layers whose gain is about one."""
    need_gpu()
    N, T = 24, 30
    agent, b, ro = make(N, T, config=short_config(13), policy_dtype=torch.bfloat16)
    for _ in range(2):
        out = ro.collect()
        assert out["memory_state"][0].dtype == torch.bfloat16
        x = ro.normalizer.normalize(out["obs"].reshape(-1, 66)).view(T, 2 * N, 66)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=again == "autocast"):
            y, state = agent.memory(x, out["dones"].reshape(T, -1).bool(), out["memory_state"])
            value = agent.get_value(y.reshape(-1, 66)).float().view(T, N, 2)
        assert float((value - out["values"]).detach().abs().max()) <= 2e-2 + 0.064
        for a, c in zip(state, ro.memory_state):
            assert a.dtype == (torch.float32 if again == "float32" else c.dtype)
            assert float((a.float() - c.float()).detach().abs().max()) <= 4 * 2.0 ** -8 * (1 + float(c.float().abs().max()))
        value.square().mean().backward()
        assert all(bool(torch.isfinite(p.grad).all()) for p in agent.memory.parameters())
    b.close()


@gpu
def test_gradients_reach_a_state_of_another_type():
    """The same as those of the state in float32, rounded to the state's type."""
    need_gpu()
    torch.manual_seed(0)
    m = SequenceMemory(channels=32).cuda()
    x = torch.randn(5, 3, 66, device="cuda")
    state = tuple(torch.randn_like(s) for s in m.init_state(3, "cuda", torch.bfloat16))
    grads = []
    for conv in (state[0], state[0].float()):
        leaves = conv.clone().requires_grad_(), state[1].clone().requires_grad_()
        grads.append(torch.autograd.grad(m(x, None, leaves)[0].sum(), leaves))
    (a, b), (c, d) = grads
    assert a.dtype == torch.bfloat16 and bool(a.any()) and torch.equal(a, c.bfloat16()) and torch.equal(b, d)


def test_the_fused_policy_refuses_an_agent_with_memory():
    from marlsoccer.policy import FusedPolicy
    with pytest.raises(ValueError, match="no memory"):
        FusedPolicy(Agent(memory=SequenceMemory()))
    fused = FusedPolicy(Agent())
    fused.agent.memory = SequenceMemory()  # given one later
    with pytest.raises(ValueError, match="no memory"):
        fused.pack()


@gpu
def test_a_replaced_state_is_captured_again():
    """A caller that puts new tensors in memory_state's place, where zeroing them was asked for: a replayed
    graph would go on from the old ones."""
    need_gpu()
    runs = []
    for graph in (False, True):
        agent, b, ro = make(24, 9, graph, short_config(7))
        outs = []
        for k in range(5):
            if k == 3:
                ro.memory_state = agent.memory.init_state(48, "cuda")
            out = ro.collect()
            outs += [out[k].clone() for k in ("obs", "actions", "values")] + [s.clone() for s in ro.memory_state + out["memory_state"]]
        runs.append(outs)
        b.close()
    assert all(torch.equal(a, c) for a, c in zip(*runs))


@gpu
def test_a_memory_that_comes_or_goes_is_refused():
    need_gpu()
    agent, b, ro = make(8, 3)
    ro.collect()
    memory, agent.memory = agent.memory, None
    with pytest.raises(ValueError, match="came or went"):
        ro.collect()
    plain = DeviceRollout(b, agent, ro.normalizer, 3)
    plain.collect()
    agent.memory = memory
    with pytest.raises(ValueError, match="came or went"):
        plain.collect()
    ro.collect()
    b.close()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_whole_update_in_a_graph(bits):
    """Memory, loss, backward and AdamW's step captured once and replayed, with new inputs and learning rates
    between, against the eager updates."""
    from marlsoccer.optim import AdamW
    need_gpu()
    T, R, runs = 12, 20, []
    for graph in (False, True):
        torch.manual_seed(0)
        m, head = SequenceMemory(channels=32).cuda(), torch.nn.Linear(66, 3).cuda()
        params = [*m.parameters(), *head.parameters()]
        opt = AdamW(params, lr=torch.full((), 1e-3, device="cuda"), max_grad_norm=0.5, state_bits=bits, rounding="stochastic" if bits == 8 else None)
        x, starts = torch.randn(T, R, 66, device="cuda"), torch.rand(T, R, device="cuda") < 0.1

        def update():
            opt.zero_grad(set_to_none=True)
            loss = head(m(x, starts)[0]).square().mean()
            loss.backward()
            opt.step()
            return loss.detach()

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            update()
        torch.cuda.current_stream().wait_stream(side)
        if graph:
            opt.zero_grad(set_to_none=True)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                captured = update()
        losses = []
        for _ in range(5):
            x.mul_(1.01)
            opt.param_groups[0]["lr"].mul_(0.9)
            if graph:
                g.replay()
            losses.append(captured.clone() if graph else update())
            torch.cuda.synchronize()
        runs.append(losses + [p.detach().clone() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


class Collector(Agent):
    """An agent with something of its own under the name: no policy's memory."""

    def __init__(self):
        super().__init__()
        self.memory = [1, 2, 3]


def test_another_kind_of_memory_is_none_of_the_policys():
    from marlsoccer.policy import FusedPolicy
    FusedPolicy(Collector())


@gpu
def test_agents_with_another_kind_of_memory_run_as_before():
    need_gpu()
    from marlsoccer import SoccerBatch
    from marlsoccer.evaluate import evaluate
    runs = []
    for cls in (Agent, Collector):
        torch.manual_seed(0)
        agent, rms = cls().cuda(), RunningMeanStd((66,), device="cuda")
        b = SoccerBatch(8, config=short_config(20))
        b.reset(seed=3)
        ro = DeviceRollout(b, agent, rms, 6, seed=5)
        assert ro.policy == "fused"
        out = ro.collect()
        assert "memory_state" not in out
        runs.append((out["values"].clone(), torch.from_numpy(evaluate(agent, rms, 4, seed=3, config=short_config(20))["returns"])))
        b.close()
    assert all(torch.equal(a, c) for a, c in zip(*runs))
