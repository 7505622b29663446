"""The gated core as it is used: projection, scan, projection with residual and AdamW together; Policy(recurrent='gated') under PPO
and A2C.  Reference: the same network in 64 bits through torch autograd."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import synth
from gated_refs import EPS

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


class Discrete(object):
    def __init__(self, n):
        self.n = n


class Box(object):
    def __init__(self, dim):
        self.shape = (dim,)


def rnd(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def core64(x, w_in, b_in, w_out, b_out, state, masks):
    H = w_out.shape[0]
    proj = x @ w_in.t() + b_in
    f, v = torch.sigmoid(proj[..., :H]), proj[..., H:]
    h, hs = state, []
    for t in range(x.shape[0]):
        h = f[t] * (masks[t][:, None] * h) + (1 - f[t]) * v[t]
        hs.append(h)
    hs = torch.stack(hs)
    return hs + F.silu(hs @ w_out.t() + b_out), h


def rel(a, b):
    a, b = a.detach().to(F64), b.detach()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize('dt', [F32, BF, HF])
@pytest.mark.parametrize('T,N,I,H', [(1, 3, 8, 16), (40, 5, 11, 32), (130, 2, 24, 20)])
def test_core_and_its_gradients(dt, T, N, I, H):
    from a2c_ppo_acktr.gated import GatedCore
    torch.manual_seed(1)
    core = GatedCore(I, H).to(DEV).to(dt)
    x, s0 = rnd(2, T, N, I, dtype=dt).requires_grad_(), rnd(3, N, H).requires_grad_()
    m = (rnd(4, T, N) < 1.3).float()
    dy, ds = rnd(5, T, N, H, dtype=dt), rnd(6, N, H)
    y, last = core(x, s0, m[..., None])
    ((y * dy).sum(dtype=F32) + (last * ds).sum()).backward()
    P = [p.detach().to(F64).requires_grad_() for p in (core.in_proj.weight, core.in_proj.bias, core.out_proj.weight, core.out_proj.bias)]
    x64, s64 = x.detach().to(F64).requires_grad_(), s0.detach().to(F64).requires_grad_()
    y64, l64 = core64(x64, *P, s64, m.to(F64))
    ((y64 * dy.to(F64)).sum() + (l64 * ds.to(F64)).sum()).backward()
    # every stage rounds its result to the storage type once (projection, states, output; and as many gradients): at most six roundings
    # of half a step each stand in a row, and a gate's derivative is a product of two rounded differences: 12 half steps of the norm
    tol = 12 * EPS[dt] + 2e-6
    assert rel(y, y64.detach()) < tol and rel(last, l64.detach()) < tol
    got = [core.in_proj.weight.grad, core.in_proj.bias.grad, core.out_proj.weight.grad, core.out_proj.bias.grad, x.grad, s0.grad]
    for i, (g, r) in enumerate(zip(got, P + [x64, s64])):
        assert g.dtype == (F32 if i == 5 else dt) and rel(g, r.grad) < 2 * tol, (i, rel(g, r.grad))


def test_steps_are_the_sequence():
    from a2c_ppo_acktr.gated import GatedCore
    core = GatedCore(12, 24).to(DEV)
    x, m = rnd(1, 9, 4, 12), (rnd(2, 9, 4) < 1.0).float()
    state = core.initial_state(4)
    with torch.no_grad():
        y, last = core(x, None, m)
    for t in range(9):
        yt = core.step(x[t], state, m[t])
        # the same arithmetic up to how steps are composed: a few roundings of values below 8
        assert float((yt - y[t]).abs().max()) < 64 * 2.0 ** -24 * 8
    assert float((state - last).abs().max()) < 64 * 2.0 ** -24 * 8


@pytest.mark.parametrize('dt', [F32, BF, HF])
@pytest.mark.parametrize('N,I,H', [(32, 512, 512), (1, 8, 16), (5, 11, 23), (3, 1, 1), (200, 40, 64), (0, 8, 8)])
def test_one_call_is_its_three_parts(dt, N, I, H):
    from a2c_ppo_acktr import ops
    wide = rnd(1, N, I + 3, dtype=dt)
    w_in, b_in = rnd(2, 2 * H, I, scale=I ** -0.5, dtype=dt), rnd(3, 2 * H, dtype=dt)
    w_out, b_out = rnd(4, H, H, scale=H ** -0.5, dtype=dt), rnd(5, H, dtype=dt)
    for x in (wide[:, :I], wide[:, 3:], wide[:, :I].contiguous()):
        for m in (None, (rnd(6, N, 1) < 0.5).float()):
            state = rnd(7, N, H)
            want_state = state.clone()
            proj = ops.linear_act_fwd(x, w_in, b_in)
            h = ops.gated_scan_step(proj[:, :H], proj[:, H:], want_state, m)
            want = ops.linear_act_fwd(h, w_out, b_out, act='silu', residual=h)
            before = state.clone()
            y, new = ops.gated_core_step(x, w_in, b_in, w_out, b_out, state, m)
            assert torch.equal(y, want) and torch.equal(new, want_state) and torch.equal(state, before)
            y, same = ops.gated_core_step(x, w_in, b_in, w_out, b_out, state, m, state)
            assert same is state and torch.equal(y, want) and torch.equal(state, want_state)


def test_one_call_captured():
    from a2c_ppo_acktr import gated, ops
    core = gated.GatedCore(24, 40).to(DEV, BF)
    x, m, state = torch.zeros(6, 24, dtype=BF, device=DEV), torch.ones(6, device=DEV), torch.zeros(6, 40, device=DEV)
    core.step(x, state.clone(), m)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with ops.graph_capture(g):
        y = core.step(x, state, m)
    state.zero_()
    eager = torch.zeros_like(state)
    for k in range(4):
        x.copy_(rnd(k, 6, 24, dtype=BF))
        m.copy_((rnd(k + 9, 6) < 1.0).float())
        want = core.step(x, eager, m)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, eager), k


def test_one_call_refusals():
    from a2c_ppo_acktr import ops
    N, I, H = 4, 8, 16
    ok = dict(x=rnd(1, N, I), w_in=rnd(2, 2 * H, I), b_in=rnd(3, 2 * H), w_out=rnd(4, H, H), b_out=rnd(5, H), state=rnd(6, N, H),
              masks=torch.ones(N, device=DEV))
    ops.gated_core_step(**ok)
    wide = torch.zeros(2 * N, H, device=DEV)
    for kw in (dict(x=rnd(1, N, I + 1)), dict(x=rnd(1, N, I, dtype=BF)), dict(w_in=rnd(2, 2 * H + 1, I)), dict(w_in=rnd(2, I, 2 * H).t()),
               dict(b_in=rnd(3, H)), dict(w_out=rnd(4, H, H + 1)), dict(b_out=rnd(5, H).half()), dict(state=rnd(6, N, H, dtype=BF)),
               dict(state=rnd(6, N + 1, H)), dict(masks=torch.ones(N, 2, device=DEV)), dict(masks=torch.ones(N, dtype=torch.bool, device=DEV)),
               dict(state=wide[:N], state_out=wide[1:N + 1]), dict(state_out=ok['w_out'][:N]), dict(x=ok['x'].cpu()), dict(state=ok['state'].cpu())):
        with pytest.raises(RuntimeError):
            ops.gated_core_step(**dict(ok, **kw))


def test_forward_and_backward_captured():
    """both passes recorded into a graph by autograd; replays follow new inputs and stay right beside eager work"""
    from a2c_ppo_acktr import gated, ops
    T, N, I, H = 70, 3, 24, 40
    core = gated.GatedCore(I, H).to(DEV)
    x, st = torch.zeros(T, N, I, device=DEV).requires_grad_(), torch.zeros(N, H, device=DEV)
    m, dy = torch.ones(T, N, device=DEV), torch.zeros(T, N, H, device=DEV)
    leaves = [x] + list(core.parameters())

    def both():
        y, last = core(x, st, m)
        return (y.detach(), last.detach()) + torch.autograd.grad(y, leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with ops.graph_capture(g):
        out = both()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(T, N, I, device=DEV))
            st.copy_(torch.randn(N, H, device=DEV))
            dy.copy_(torch.randn(T, N, H, device=DEV))
            m.copy_((torch.rand(T, N, device=DEV) > 0.1).float())
        want = [t.clone() for t in both()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_autograd_corners():
    from a2c_ppo_acktr.gated import gated_scan, linear_act
    # a residual that is broadcast, an input used twice, a gradient that is expanded, no gradient for a part
    x, w = rnd(1, 6, 8).requires_grad_(), rnd(2, 8, 8, scale=0.3).requires_grad_()
    r = rnd(3, 8).requires_grad_()
    linear_act(x, w, None, 'tanh', r.expand(6, 8)).sum().backward()
    assert torch.equal(r.grad, torch.full((8,), 6.0, device=DEV))
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    torch.tanh(x64 @ w64.t()).sum().backward()
    assert rel(x.grad, x64.grad) < 1e-5 and rel(w.grad, w64.grad) < 1e-5
    g = rnd(4, 5, 2, 8).requires_grad_()
    out, last = gated_scan(g, g)                             # gate and value the same tensor
    last.sum().backward()                                    # nothing reaches the states
    g64 = g.detach().double().requires_grad_()
    h = torch.zeros(2, 8, dtype=F64, device=DEV)
    for t in range(5):
        f = torch.sigmoid(g64[t])
        h = f * h + (1 - f) * g64[t]
    h.sum().backward()
    assert rel(g.grad, g64.grad) < 1e-5
    with torch.no_grad():
        assert linear_act(x.t()[:6, :6], w[:, :6].contiguous()).shape == (6, 8)         # a transposed input is taken
    y = linear_act(x, w, None, 'silu')
    gx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()                                  # no second derivatives, and no wrong ones
    with pytest.raises(RuntimeError):
        linear_act(x, w, None, None, r)


def test_writes_in_place_are_seen_by_autograd():
    """a pending backward pass whose saved tensors were overwritten raises, as it does for torch's own in-place operations"""
    from a2c_ppo_acktr import algo, ops
    from a2c_ppo_acktr.gated import GatedCore, gated_scan, linear_act
    core, x, state = GatedCore(8, 16).to(DEV), rnd(1, 5, 3, 8), rnd(2, 3, 16)
    proj = rnd(3, 3, 32)
    # the state that a sequence started from, by each of the calls that take a step
    for step in (lambda s: core.step(x[0], s), lambda s: ops.gated_scan_step(proj[:, :16], proj[:, 16:], s),
                 lambda s: ops.gated_core_step(x[0], core.in_proj.weight, core.in_proj.bias, core.out_proj.weight, core.out_proj.bias, rnd(4, 3, 16), None, s)):
        y, _ = core(x, state)
        with torch.no_grad():
            step(state)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()
    # weights, and 16-bit copies of them
    for w, opt in ((core.out_proj.weight, lambda w: algo.AdamW([w], lr=1e-3, grads=[torch.ones_like(w)])),
                   (rnd(5, 4, 8, dtype=BF).requires_grad_(), lambda w: algo.AdamW([w.detach().float()], lr=1e-3, grads=[torch.ones_like(w)], copies=[w]))):
        a = rnd(6, 7, w.shape[1], dtype=w.dtype).requires_grad_()
        y = linear_act(a, w)
        opt(w).step()
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            y.sum().backward()


@pytest.mark.parametrize('T,N', [(0, 3), (5, 0), (0, 0)])
def test_no_steps_or_no_sequences(T, N):
    from a2c_ppo_acktr.gated import GatedCore
    core = GatedCore(8, 16).to(DEV, BF)
    x, s0 = torch.zeros(T, N, 8, dtype=BF, device=DEV).requires_grad_(), rnd(1, N, 16).requires_grad_()
    y, last = core(x, s0, torch.ones(T, N, 1, device=DEV))
    assert y.shape == (T, N, 16) and last.shape == (N, 16) and (T or torch.equal(last, s0))
    (y.sum(dtype=F32) + last.sum()).backward()
    assert x.grad.shape == x.shape and (T or torch.equal(s0.grad, torch.ones_like(s0)))
    assert all(p.grad is not None and not p.grad.any() for p in core.parameters())
    assert core.step(torch.zeros(N, 8, dtype=BF, device=DEV), last.detach()).shape == (N, 16)


@pytest.mark.parametrize('dt', [BF, F32])
def test_gradients_into_rows_of_wider_tensors(dt):
    from a2c_ppo_acktr import ops
    M, N, K = 70, 40, 51
    x, w, dy = rnd(1, M, K, dtype=dt), rnd(2, N, K, dtype=dt), rnd(3, M, N, dtype=dt)
    want = ops.linear_act_bwd(dy, x, w)
    big, vec = torch.full((M + 2, 2 * K + 3), 5.0, dtype=dt, device=DEV), torch.full((N + 2,), 5.0, dtype=dt, device=DEV)
    ops.linear_act_bwd(dy, x, w, dx=big[1:M + 1, K:2 * K], db=vec[1:N + 1])
    assert torch.equal(big[1:M + 1, K:2 * K], want[0]) and torch.equal(vec[1:N + 1], want[2])
    big[1:M + 1, K:2 * K] = 5
    vec[1:N + 1] = 5
    assert bool((big == 5).all()) and bool((vec == 5).all())


def test_streams_of_their_own():
    """training steps of two cores on two streams at once, and what they give in turn on one"""
    from a2c_ppo_acktr import algo
    from a2c_ppo_acktr.gated import GatedCore
    T, N, I, H = 300, 4, 40, 64

    def make(seed):
        torch.manual_seed(seed)
        core = GatedCore(I, H).to(DEV, BF)
        masters = [p.detach().float() for p in core.parameters()]
        opt = algo.AdamW(masters, lr=1e-3, copies=list(core.parameters()), max_grad_norm=0.5, state_bits=8, seed=seed)
        return core, masters, opt, rnd(seed, T, N, I, dtype=BF), (rnd(seed + 9, T, N) < 1.5).float()

    def train(core, masters, opt, x, m):
        y, last = core(x, None, m)
        for p, g in zip(core.parameters(), torch.autograd.grad((y.float() ** 2).mean() + last.mean(), list(core.parameters()))):
            p.grad = g
        opt.step()
    want = []
    for seed in (1, 2):
        job = make(seed)
        for _ in range(4):
            train(*job)
        want.append([p.clone() for p in job[1]])
    jobs, streams = [make(1), make(2)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        for job, st in zip(jobs, streams):
            with torch.cuda.stream(st):
                train(*job)
    torch.cuda.synchronize()
    for job, w in zip(jobs, want):
        assert all(torch.equal(p, q) for p, q in zip(job[1], w))


def test_given_outputs_are_marked_as_changed():
    from a2c_ppo_acktr import ops
    x, w, dy = rnd(1, 6, 8), rnd(2, 4, 8), rnd(3, 6, 4)
    new = lambda *s: torch.zeros(*s, device=DEV)
    out, pre, dx, dw, db = new(6, 4), new(6, 4), new(6, 8), new(4, 8), new(4)
    ops.linear_act_fwd(x, w, act='tanh', out=out, pre=pre)
    ops.linear_act_bwd(dy, x, w, pre=pre, act='tanh', dx=dx, dw=dw, db=db)
    g, v, so, dg, dv = rnd(4, 5, 2, 8), rnd(5, 5, 2, 8), new(5, 2, 8), new(5, 2, 8), new(5, 2, 8)
    _, _, saved = ops.gated_scan_fwd(g, v, out=so, save=True)
    ops.gated_scan_bwd(v, g, v, saved=saved, dgate=dg, dvalue=dv)
    state, one = new(2, 8), new(2, 8)
    ops.gated_scan_step(g[0], v[0], state, out=one)
    assert [t._version for t in (out, pre, dx, dw, db, so, dg, dv, state, one)] == [1] * 10
    assert [t._version for t in (x, w, dy, g, v)] == [0] * 5
    with torch.inference_mode():                             # (their versions are not counted)
        s = torch.zeros(2, 8, device=DEV)
        ops.gated_scan_step(g[0], v[0], s)
    assert torch.equal(s, state)


@pytest.mark.parametrize('bits', [32, 8])
def test_mixed_precision_training(bits):
    """bf16 weights and gradients, fp32 masters, AdamW writing both: three steps of a small core against the same steps in 64 bits on
    the weights the layer really used"""
    from a2c_ppo_acktr import algo
    from a2c_ppo_acktr.gated import GatedCore
    torch.manual_seed(2)
    T, N, I, H = 24, 4, 16, 32
    core = GatedCore(I, H).to(DEV)
    masters = [p.detach().clone() for p in core.parameters()]
    core.to(BF)
    weights = list(core.parameters())
    hp = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    opt = algo.AdamW(masters, copies=weights, state_bits=bits, max_grad_norm=1.0, seed=4, **hp)
    x, m, tgt = rnd(3, T, N, I, dtype=BF), (rnd(4, T, N) < 1.5).float(), rnd(5, T, N, H)
    ref = [p.double() for p in masters]
    mom = [[torch.zeros_like(p), torch.zeros_like(p)] for p in ref]
    for k in range(1, 4):
        opt.zero_grad(set_to_none=True)
        y, _ = core(x, None, m)
        ((y.float() - tgt) ** 2).mean().backward()
        P = [p.detach().double().requires_grad_() for p in weights]
        y64, _ = core64(x.double(), *P, torch.zeros(N, H, dtype=F64, device=DEV), m.double())
        ((y64 - tgt.double()) ** 2).mean().backward()
        for p, r in zip(weights, P):
            assert rel(p.grad, r.grad) < 30 * EPS[BF]        # as in test_core_and_its_gradients, and the loss' own bf16 seed
        grads = [p.grad.double() for p in weights]           # (the step is checked on the gradients that it was given)
        opt.step()
        norm = float(sum((g * g).sum() for g in grads)) ** 0.5
        c = min(1.0, 1.0 / (norm + 1e-6))
        for i, g in enumerate(grads):
            a, b = mom[i]
            a.mul_(0.9).add_(0.1 * c * g), b.mul_(0.99).add_(0.01 * (c * g) ** 2)
            ref[i] = ref[i] * (1 - 1e-2 * 0.1) - 1e-2 / (1 - 0.9 ** k) * a / (b.sqrt() / (1 - 0.99 ** k) ** 0.5 + 1e-8)
            got = masters[i].double()
            if bits == 32:
                assert float((got - ref[i]).abs().max()) < 1e-2 * 1e-4 + 1e-6
            elif k == 1:                                     # the first step does not depend on how the moments are kept
                assert float((got - ref[i]).abs().max()) < 1e-2 * 1e-4 + 1e-6
            assert torch.equal(weights[i].detach(), masters[i].to(BF))


def make_policy(kind, seed=3):
    from a2c_ppo_acktr.model import Policy
    torch.manual_seed(seed)
    pol = Policy((4, 84, 84), Discrete(6), base_kwargs={'recurrent': 'gated'}) if kind == 'cnn' else \
        Policy((11,), Box(3), base_kwargs={'recurrent': 'gated'})
    return pol.to(DEV)


def policy64(pol, obs, act, hxs, masks, T, N):
    """value, log-probability, entropy of a gated policy in 64 bits, with leaves to differentiate"""
    P = {n: p.detach().to(F64).requires_grad_() for n, p in pol.named_parameters()}
    x = obs.to(F64)
    core = lambda q: core64(q.view(T, N, -1), P['base.core.in_proj.weight'], P['base.core.in_proj.bias'], P['base.core.out_proj.weight'],
                            P['base.core.out_proj.bias'], hxs.to(F64), masks.to(F64).view(T, N))
    lin = lambda q, n: q @ P[n + '.weight'].t() + P[n + '.bias']
    if 'base.main.0.weight' in P:
        c = lambda q, i, s: F.relu(F.conv2d(q, P['base.main.%d.weight' % i], P['base.main.%d.bias' % i], stride=s))
        q = c(c(c(x / 255.0, 0, 4), 2, 2), 4, 1).flatten(1)
        y, last = core(F.relu(lin(q, 'base.main.7')))
        y = y.reshape(T * N, -1)
        value, logits = lin(y, 'base.critic_linear'), lin(y, 'dist.linear')
        d = torch.distributions.Categorical(logits=logits)
        return P, value, d.log_prob(act.view(-1)).view(-1, 1), d.entropy().mean(), last
    y, last = core(x)
    y = y.reshape(T * N, -1)
    tower = lambda n: torch.tanh(lin(torch.tanh(lin(y, 'base.%s.0' % n)), 'base.%s.2' % n))
    value, mean = lin(tower('critic'), 'base.critic_linear'), lin(tower('actor'), 'dist.fc_mean')
    d = torch.distributions.Normal(mean, P['dist.logstd._bias'].view(1, -1).exp().expand_as(mean))
    return P, value, d.log_prob(act.to(F64)).sum(-1, keepdim=True), d.entropy().sum(-1).mean(), last


@pytest.mark.parametrize('kind,T,N', [('mlp', 40, 3), ('mlp', 1, 5), ('cnn', 6, 3)])
def test_policy_gradients(kind, T, N):
    pol = make_policy(kind)
    H = pol.recurrent_hidden_state_size
    obs = rnd(1, T * N, 11) if kind == 'mlp' else (rnd(1, T * N, 4, 84, 84).abs() * 80).clamp(max=255).round()
    act = rnd(2, T * N, 3) if kind == 'mlp' else torch.arange(T * N, device=DEV).view(-1, 1) % 6
    hxs, masks = rnd(3, N, H, scale=0.5), (rnd(4, T * N, 1) < 1.0).float()
    v, lp, ent, h = pol.evaluate_actions(obs, hxs, masks, act)
    cv, cl = rnd(5, T * N, 1), rnd(6, T * N, 1)
    pol.zero_grad()
    ((v * cv).sum() + (lp * cl).sum() + ent).backward()
    P, v64, lp64, e64, h64 = policy64(pol, obs, act, hxs, masks, T, N)
    ((v64 * cv.to(F64)).sum() + (lp64 * cl.to(F64)).sum() + e64).backward()
    for a, b in ((v, v64), (lp, lp64), (ent, e64), (h, h64)):
        assert rel(a.detach(), b.detach()) < 1e-5
    for n, p in pol.named_parameters():
        # fp32 sums of up to T N 400 terms; a ReLU gate within rounding of zero may go the other way on the convolutions
        assert rel(p.grad, P[n].grad) < (1e-3 if kind == 'cnn' else 5e-5), (n, rel(p.grad, P[n].grad))
    # acting: single steps reproduce the sequence
    s = hxs
    for t in range(T):
        sl = slice(t * N, (t + 1) * N)
        vt, _, _, s2 = pol.act(obs[sl], s, masks[sl], deterministic=True)
        assert torch.equal(vt, pol.get_value(obs[sl], s, masks[sl]))
        np.testing.assert_allclose(vt.cpu().numpy(), v[sl].detach().cpu().numpy(), rtol=1e-4, atol=1e-5)
        s = s2
    np.testing.assert_allclose(s.cpu().numpy(), h.cpu().numpy(), rtol=1e-4, atol=1e-5)


def make_storage(kind, T, N, H, seed=0):
    from a2c_ppo_acktr.storage import RolloutStorage
    space = Discrete(6) if kind == 'cnn' else Box(3)
    shape = (4, 84, 84) if kind == 'cnn' else (11,)
    ro = synth.make_rollouts(T, N, shape, 'discrete' if kind == 'cnn' else 'box', 6 if kind == 'cnn' else 3, salt=41 + seed)
    rs = RolloutStorage(T, N, shape, space, H)
    for k in ('obs', 'rewards', 'value_preds', 'returns', 'action_log_probs', 'actions', 'masks', 'bad_masks'):
        getattr(rs, k).copy_(torch.from_numpy(np.ascontiguousarray(ro[k])))
    rs.to(DEV)
    rs.compute_returns(torch.from_numpy(ro['next_value']).to(DEV), True, 0.99, 0.95, True)
    return rs


@pytest.mark.parametrize('kind,T,N,nmb', [('mlp', 24, 6, 3), ('cnn', 5, 4, 2)])
@pytest.mark.parametrize('opt', [dict(), dict(weight_decay=0.05), dict(weight_decay=0.05, state_bits=8)])
def test_ppo_updates(kind, T, N, nmb, opt):
    """four updates, the later ones replayed from a captured graph, equal the same updates launch by launch"""
    from a2c_ppo_acktr import algo
    res = []
    for graph in (True, False):
        pol = make_policy(kind)
        p0 = pol.flat_params.clone()
        agent = algo.PPO(pol, 0.2, 2, nmb, 0.5, 0.01, lr=3e-4, eps=1e-5, max_grad_norm=0.5, **opt)
        agent.use_graph = graph
        rs = make_storage(kind, T, N, pol.recurrent_hidden_state_size)
        losses = []
        for it in range(4):
            torch.manual_seed(100 + it)
            losses.append(agent.update(rs))
        assert (agent._rgraph is not None) == graph
        assert all(np.isfinite(losses).ravel()) and not torch.equal(pol.flat_params, p0)
        assert agent.optimizer.step_count == 4 * 2 * nmb
        res.append((pol.flat_params.clone(), losses))
    assert torch.equal(res[0][0], res[1][0]) and np.array_equal(res[0][1], res[1][1])


@pytest.mark.parametrize('kind', ['mlp', 'cnn'])
def test_ppo_adamw_without_recurrence(kind):
    """feed-forward policies with AdamW, against the flat Adam where both do the same (no decay)"""
    from a2c_ppo_acktr import algo
    from a2c_ppo_acktr.model import Policy
    out = []
    for opt in (dict(), dict(weight_decay=0.0)):
        torch.manual_seed(5)
        pol = (Policy((11,), Box(3)) if kind == 'mlp' else Policy((4, 84, 84), Discrete(6))).to(DEV)
        agent = algo.PPO(pol, 0.2, 2, 2, 0.5, 0.01, lr=3e-4, eps=1e-5, max_grad_norm=0.5, **opt)
        rs = make_storage(kind, 8, 4, 1)
        for it in range(3):
            torch.manual_seed(100 + it)
            agent.update(rs)
        out.append(pol.flat_params.clone())
    # 12 steps of at most lr each; the two kernels round differently, and a step's direction follows the sign of tiny gradients
    assert float((out[0] - out[1]).abs().max()) < 12 * 3e-4 * 0.5 and rel(out[0], out[1].double()) < 1e-4


@pytest.mark.parametrize('rec', ['gated', False])
def test_ppo_adamw_clip_changes(rec):
    """the agent's clip norm may be None, and may change between updates; replays and plain launches agree"""
    from a2c_ppo_acktr import algo
    from a2c_ppo_acktr.model import Policy
    res = []
    for graph in (True, False):
        torch.manual_seed(5)
        pol = Policy((11,), Box(3), base_kwargs={'recurrent': rec}).to(DEV)
        agent = algo.PPO(pol, 0.2, 2, 2, 0.5, 0.01, lr=3e-4, eps=1e-5, max_grad_norm=None, weight_decay=0.01)
        agent.use_graph = graph
        rs = make_storage('mlp', 8, 4, pol.recurrent_hidden_state_size)
        for it, clip in enumerate((None, None, None, 0.1, 0.1, 0.1, None, None, None)):
            agent.max_grad_norm = clip
            agent.optimizer.param_groups[0]['lr'] = 3e-4 / (it + 1)
            torch.manual_seed(100 + it)
            agent.update(rs)
        res.append(pol.flat_params.clone())
    assert torch.equal(*res)


def test_a2c_updates():
    from a2c_ppo_acktr import algo
    for kind, T, N in (('mlp', 7, 4), ('cnn', 5, 3)):
        pol = make_policy(kind)
        p0 = pol.flat_params.clone()
        agent = algo.A2C_ACKTR(pol, 0.5, 0.01, lr=7e-4, eps=1e-5, alpha=0.99, max_grad_norm=0.5)
        rs = make_storage(kind, T, N, pol.recurrent_hidden_state_size)
        for _ in range(3):
            assert all(np.isfinite(agent.update(rs)))
        assert not torch.equal(pol.flat_params, p0) and bool(pol.flat_params.isfinite().all())
    with pytest.raises(NotImplementedError):
        algo.A2C_ACKTR(make_policy('mlp'), 0.5, 0.01, acktr=True)


def test_checkpoint(tmp_path):
    pol = make_policy('mlp')
    obs, hxs, m = rnd(1, 4, 11), rnd(2, 4, 64), torch.ones(4, 1, device=DEV)
    v = pol.get_value(obs, hxs, m)
    torch.save([pol, None], tmp_path / 'p.pt')
    p2, _ = torch.load(tmp_path / 'p.pt', weights_only=False)        # written two lines above
    assert torch.equal(p2.get_value(obs, hxs, m), v)
