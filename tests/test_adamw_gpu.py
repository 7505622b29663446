"""algo.AdamW over many tensors against 64-bit and plain fp32 evaluations."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E32 = 2.0 ** -24
EPS = {F32: 2.0 ** -24, HF: 2.0 ** -11, BF: 2.0 ** -8}
SHAPES = [(1,), (3,), (255,), (256,), (257,), (64, 33), (2048,), (2049,), (5, 4099), (0,), (70, 100)]
HP = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)


def rnd(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def make(shapes=SHAPES, pdt=F32, gdt=F32, cdt=None, odd=False, seed=0):
    def alloc(s, dt, k, scale):
        n = math.prod(s)
        if odd:                                             # tensors that start anywhere
            return rnd(seed + k, n + 3, scale=scale, dtype=dt)[1 + k % 3:1 + k % 3 + n].view(s)
        return rnd(seed + k, *s, scale=scale, dtype=dt)
    ps = [alloc(s, pdt, 10 * i, 0.5) for i, s in enumerate(shapes)]
    gs = [alloc(s, gdt, 10 * i + 1, 0.1) for i, s in enumerate(shapes)]
    cs = [alloc(s, cdt, 10 * i + 2, 1.0) if cdt is not None and i % 3 != 1 else None for i, s in enumerate(shapes)]
    return ps, gs, cs


def ref_steps(ps, grads, clip, hp=HP):
    """parameters, moments after each step's gradients, in 64 bits"""
    b1, b2 = hp['betas']
    ps = [p.to(F64) for p in ps]
    ms, vs = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    for t, gs in enumerate(grads, 1):
        gs = [g.to(F64) for g in gs]
        if clip:
            norm = math.sqrt(sum(float((g * g).sum()) for g in gs))
            gs = [g * min(1.0, clip / (norm + 1e-6)) for g in gs]
        for i, g in enumerate(gs):
            ms[i] = b1 * ms[i] + (1 - b1) * g
            vs[i] = b2 * vs[i] + (1 - b2) * g * g
            ps[i] = ps[i] * (1 - hp['lr'] * hp['weight_decay']) - hp['lr'] / (1 - b1 ** t) * ms[i] / (
                vs[i].sqrt() / math.sqrt(1 - b2 ** t) + hp['eps'])
    return ps, ms, vs


def moments_of(opt, shapes):
    m, v = opt.moments()
    return [[b[o:o + math.prod(s)].view(s) for o, s in zip(opt.offsets(), shapes)] for b in (m, v)]


@pytest.mark.parametrize('odd', [False, True])
@pytest.mark.parametrize('clip', [None, 0.5])
@pytest.mark.parametrize('gdt', [F32, BF, HF])
def test_fp32_moments(gdt, clip, odd):
    from a2c_ppo_acktr import algo
    steps = 4
    ps, gs, cs = make(gdt=gdt, cdt=BF, odd=odd)
    p0 = [p.clone() for p in ps]
    opt = algo.AdamW(ps, grads=gs, copies=cs, max_grad_norm=clip, **HP)
    hist = []
    for k in range(steps):
        for i, g in enumerate(gs):
            g.copy_(rnd(500 + 50 * k + i, *g.shape, scale=0.1))
        hist.append([g.clone() for g in gs])
        opt.step()
    rp, rm, rv = ref_steps(p0, hist, clip)
    m, v = moments_of(opt, SHAPES)
    amax = [torch.stack([h[i].to(F64).abs() for h in hist]).amax(0) for i in range(len(SHAPES))]
    for i in range(len(SHAPES)):
        # every step rounds a handful of times: 8 roundings of a moment, of g at most; the parameter moves by at most
        # lr / (1 - b1) a step with a relative error of 16 roundings and of sqrt(v), and is itself rounded three times a step
        tm = 8 * steps * E32 * amax[i]
        tv = 8 * steps * E32 * amax[i] ** 2
        tp = steps * (3 * E32 * (rp[i].abs() + 0.1) + 64 * E32 * HP['lr'] / (1 - HP['betas'][0]))
        assert bool(((m[i].to(F64) - rm[i]).abs() <= tm).all()) and bool(((v[i].to(F64) - rv[i]).abs() <= tv).all()), i
        assert bool(((ps[i].to(F64) - rp[i]).abs() <= tp).all()), (i, float((ps[i].to(F64) - rp[i]).abs().max()))
        if cs[i] is not None:
            assert torch.equal(cs[i], ps[i].to(BF))
    assert opt.steps_done() == steps


@pytest.mark.parametrize('pdt', [BF, HF])
def test_16_bit_parameters(pdt):
    from a2c_ppo_acktr import algo
    ps, gs, _ = make(pdt=pdt, gdt=pdt)
    p0 = [p.clone() for p in ps]
    algo.AdamW(ps, grads=gs, **HP).step()
    rp, _, _ = ref_steps(p0, [gs], None)
    for p, r in zip(ps, rp):
        assert bool(((p.to(F64) - r).abs() <= EPS[pdt] * r.abs() + 1e-6).all())      # one rounding; fp32 inside


# more chunks (of 2048) than the update's workgroups sum for themselves, around the norm's 1024 workgroups with two chunks each
LONG = [[(1025 * 2048 - 700,), (300,)], [(1200, 1700), (3,), (2048, 1031), (77,)], [(5000, 2048), (1,), (65537,)]]


@pytest.mark.parametrize('odd', [False, True])
@pytest.mark.parametrize('shapes', LONG)
@pytest.mark.parametrize('gdt', [F32, BF])
def test_clipped_lists_of_many_chunks(gdt, shapes, odd):
    """the norm of a long list: its own launch finishes it, step after step, captured too"""
    from a2c_ppo_acktr import algo, ops
    steps, clip, runs = 4, 0.5, []
    for captured in (False, True, False):
        ps, gs, cs = make(shapes, gdt=gdt, cdt=BF, odd=odd)
        p0 = [p.clone() for p in ps]
        opt = algo.AdamW(ps, grads=gs, copies=cs, max_grad_norm=clip, **HP)
        graph, hist = None, []
        for k in range(steps):
            for i, g in enumerate(gs):
                g.copy_(rnd(500 + 50 * k + i, *g.shape, scale=0.1 + 0.2 * k))
            hist.append([g.clone() for g in gs])
            if captured and k == 1:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with ops.graph_capture(graph):
                    opt.step()
            opt.step() if graph is None else graph.replay()
            torch.cuda.synchronize()
        assert opt.steps_done() == steps
        runs.append([p.clone() for p in ps] + list(opt.moments()))
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*runs))
    rp, rm, rv = ref_steps(p0, hist, clip)
    m, v = moments_of(opt, shapes)
    for i in range(len(shapes)):                             # (as in test_fp32_moments)
        amax = torch.stack([h[i].to(F64).abs() for h in hist]).amax(0)
        tp = steps * (3 * E32 * (rp[i].abs() + 0.1) + 64 * E32 * HP['lr'] / (1 - HP['betas'][0]))
        assert bool(((m[i].to(F64) - rm[i]).abs() <= 8 * steps * E32 * amax).all()), i
        assert bool(((v[i].to(F64) - rv[i]).abs() <= 8 * steps * E32 * amax ** 2).all()), i
        assert bool(((ps[i].to(F64) - rp[i]).abs() <= tp).all()), (i, float((ps[i].to(F64) - rp[i]).abs().max()))
        if cs[i] is not None:
            assert torch.equal(cs[i], ps[i].to(BF))


@pytest.mark.parametrize('shapes', LONG)
def test_clipped_8_bit_lists_of_many_chunks(shapes):
    """the first step does not depend on how moments are kept; later ones repeat bit for bit, and a clip far above the norm is none"""
    from a2c_ppo_acktr import algo
    runs = []
    for clip in (0.5, 0.5, 1e9, None):
        ps, gs, _ = make(shapes)
        p0 = [p.clone() for p in ps]
        opt = algo.AdamW(ps, grads=gs, max_grad_norm=clip, state_bits=8, seed=7, **HP)
        opt.step()
        if clip != 1e9:
            rp, _, _ = ref_steps(p0, [gs], clip)
            for p, r in zip(ps, rp):
                assert bool(((p.to(F64) - r).abs() <= 3 * E32 * (r.abs() + 0.1) + 64 * E32 * HP['lr'] / (1 - HP['betas'][0])).all())
        opt.step(), opt.step()
        runs.append([p.clone() for p in ps] + list(opt.moments()))
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1])) and all(torch.equal(a, b) for a, b in zip(runs[2], runs[3]))
    assert not torch.equal(runs[0][0], runs[2][0])


# ------------------------------------------------------------------------------------------------ 8-bit moments, restated
def mix(x):
    x = (x ^ (x >> 16)) * 0x7feb352d & 0xffffffff
    x = (x ^ (x >> 15)) * 0x846ca68b & 0xffffffff
    return x ^ (x >> 16)


def table(top, signed):
    """value of every code for a scale of 1, from the definition"""
    out = []
    for c in range(256):
        e, k = (c >> 3) & top, c & 7
        mag = (1 + k / 8) * 2.0 ** (e - top) if e else k / 8 * 2.0 ** (1 - top)
        out.append(-mag if signed and c & 128 else mag)
    return torch.tensor(out, dtype=F64, device=DEV)


def encode(x, rnd20, top, signed):
    """codes and scales by search in the table: x / scale lies between two neighbouring values; the upper one is taken when the
    random number is at least what is missing to it"""
    x = x.view(-1, 256)
    most = x.abs().amax(1, keepdim=True)
    # (a power of two by its exponent field: the device's pow, and with it ldexp, is not exact)
    scale = torch.where(most > 0, (((most.view(torch.int32) >> 23) + 1) << 23).view(F32), torch.zeros_like(most)).to(F64)
    y = torch.where(scale > 0, x.to(F64).abs() / scale, torch.zeros_like(x, dtype=F64))
    grid = table(top, False)[:128 if signed else 256]
    lo = (torch.searchsorted(grid, y.contiguous(), right=True) - 1).clamp(0, len(grid) - 2)
    frac = (y - grid[lo]) / (grid[lo + 1] - grid[lo])
    up = (torch.floor(frac * 2 ** 20 + 1e-9) + rnd20.view_as(frac)) >= 2 ** 20
    code = lo + up
    if not signed:
        code = torch.where((code == 0) & (y > 0), torch.ones_like(code), code)
    return torch.where((x < 0), code + 128, code) if signed else code, scale


@pytest.mark.parametrize('clip', [None, 0.5])
def test_8_bit_moments(clip):
    """bit for bit: the fp32 moments of every step, formed from the decoded ones in the stated order, encoded by table search"""
    from a2c_ppo_acktr import algo
    seed = 77
    ps, gs, cs = make(gdt=F32)
    for i, g in enumerate(gs):                              # magnitudes over six orders within a block
        g.mul_(torch.exp(3 * rnd(900 + i, *g.shape)))
    opt = algo.AdamW(ps, grads=gs, max_grad_norm=clip, state_bits=8, seed=seed, **HP)
    offs = opt.offsets()
    total = opt.mom1.numel()
    m, v = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
    inside = torch.zeros(total, dtype=torch.bool, device=DEV)
    b1, b2 = HP['betas']
    for t in range(1, 4):
        flat = torch.zeros(total, device=DEV)
        for o, g in zip(offs, gs):
            flat[o:o + g.numel()] = g.reshape(-1)
            inside[o:o + g.numel()] = True
        if clip:
            norm = flat.double().square().sum().sqrt()
            flat = flat * (clip / (norm + 1e-6)).clamp(max=1).float()
        m = m * b1 + flat * (1 - b1)
        v = v * b2 + (flat * flat) * (1 - b2)
        opt.step()
        r = mix(torch.arange(total, device=DEV) ^ mix((seed + t * 0x9e3779b9) & 0xffffffff))
        cm, sm = encode(m, r & 0xfffff, 15, True)
        cv, sv = encode(v, r >> 12, 31, False)
        for got, want in ((opt.mom1, cm), (opt.mom2, cv)):
            g, w = got.long().view(-1), want.view(-1)
            # below a scale's smallest exponent the fp32 sum y + 2^-14 rounds y to 2^-37: a draw within that of a border may go the
            # other way.  Of 2^20 draws that is one in 2^17 or so; the codes differ by one there.
            off = (g != w)
            assert int(off.sum()) <= 3 and int((g - w).abs().max()) <= 1, (t, int(off.sum()))
        s = opt.scales.view(-1, 2).double()
        assert torch.equal(s[:, :1], sm) and torch.equal(s[:, 1:], sv)
        gm, gv = opt.moments()
        tm, tv = table(15, True), table(31, False)
        assert torch.equal(gm.double(), (tm[opt.mom1.long()].view(-1, 256) * s[:, :1]).view(-1))
        assert torch.equal(gv.double(), (tv[opt.mom2.long()].view(-1, 256) * s[:, 1:]).view(-1))
        assert not bool(gm[~inside].any()) and not bool(gv[~inside].any())
        assert bool((gv[v > 0] > 0).all())                   # a positive v stays positive
        m, v = gm, gv
        for i, g in enumerate(gs):
            g.copy_(rnd(700 + 20 * t + i, *g.shape, scale=0.1))


def test_8_bit_rounding_keeps_the_mean():
    """one value held in 65536 places: the mean of its codes' values is the value, within six standard deviations of the draw
    (spacing / 2 each)"""
    from a2c_ppo_acktr import algo
    n = 65536
    for x in (0.3, 0.01234, 1.7e-4, 3e-6):
        p, g = torch.zeros(n, device=DEV), torch.full((n,), x, device=DEV)
        g[::256] = 1.0                                       # every block's largest
        opt = algo.AdamW([p], grads=[g], state_bits=8, seed=3, **HP)
        opt.step()
        m, v = opt.moments()
        keep = torch.ones(n, dtype=torch.bool, device=DEV)
        keep[::256] = False
        for got, want, top in ((m, (1 - HP['betas'][0]) * x, 15), (v, (1 - HP['betas'][1]) * x * x, 31)):
            vals = got[keep].double()
            lo, hi = float(vals.min()), float(vals.max())
            if top == 31 and want < 2.0 ** -39:              # below the smallest code (2^-33 of the scale 2^-6): held there, never at 0
                assert lo == hi == 2.0 ** -39
                continue
            assert lo <= want * (1 + 1e-6) and hi >= want * (1 - 1e-6) and len(vals.unique()) <= 2
            assert abs(float(vals.mean()) - want) <= 6 * (hi - lo) / 2 / n ** 0.5 + 1e-6 * want, (x, top)


def test_8_bit_follows_32_bit():
    """over many steps the parameters stay near the 32-bit ones: the codes' spacing is at most an eighth, so a step's size is off by an
    eighth (m) and a sixteenth (v) at most, and by a fraction of that on average"""
    from a2c_ppo_acktr import algo
    res = []
    for bits in (32, 8):
        p, g = rnd(1, 5000, scale=0.5), torch.zeros(5000, device=DEV)
        p0 = p.clone()
        opt = algo.AdamW([p], grads=[g], state_bits=bits, seed=1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
        for k in range(200):
            g.copy_(0.1 + rnd(30 + k, 5000, scale=0.05) * torch.linspace(0.1, 3, 5000, device=DEV))
            opt.step()
        res.append(p - p0)
    assert float((res[0] - res[1]).norm() / res[0].norm()) < 0.125 + 0.0625


def test_values_that_are_not_finite():
    from a2c_ppo_acktr import algo
    for bits in (32, 8):
        p, q, g, h = rnd(1, 700), rnd(2, 50), rnd(3, 700, scale=0.1), rnd(4, 50, scale=0.1)
        g[300] = float('nan')
        opt = algo.AdamW([p, q], grads=[g, h], state_bits=bits, **HP)
        opt.step()
        assert bool(p[300].isnan()) and bool(q.isfinite().all()) and int(p.isnan().sum()) == 1
        m, _ = opt.moments()
        assert bool(m[300].isnan())
        opt.step()
        assert bool(p[:256].isfinite().all()) and bool(q.isfinite().all())
        opt = algo.AdamW([p, q], grads=[g, h], state_bits=bits, max_grad_norm=1.0, **HP)
        opt.step()
        assert bool(q.isnan().all())                         # the norm is not a number


def test_gradients_from_the_parameters():
    from a2c_ppo_acktr import algo
    ps = [rnd(i, 40, 5).requires_grad_() for i in range(3)]
    copies = [p.detach().to(BF).requires_grad_() for p in ps]
    opt = algo.AdamW([p.detach() for p in ps], copies=copies, **HP)
    with pytest.raises(RuntimeError):
        opt.step()
    for k in range(2):                                       # fresh gradient tensors every step
        for i, c in enumerate(copies):
            c.grad = rnd(90 + 3 * k + i, 40, 5, dtype=BF)
        before = [p.detach().clone() for p in ps]
        opt.step()
        assert all(not torch.equal(p.detach(), b) for p, b in zip(ps, before))
        assert all(torch.equal(c.detach(), p.detach().to(BF)) for p, c in zip(ps, copies))
    opt.zero_grad()
    assert all(not c.grad.any() for c in copies)


def test_hyperparameters_change():
    from a2c_ppo_acktr import algo
    p, g = rnd(1, 1000), rnd(2, 1000)
    opt = algo.AdamW([p], grads=[g], **HP)
    opt.step()
    q = p.clone()
    opt.param_groups[0]['lr'] = 0.0
    opt.step()
    assert torch.equal(p, q)
    opt.param_groups[0]['lr'] = -1.0
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.parametrize('bits', [32, 8])
def test_state_round_trip(bits, tmp_path):
    from a2c_ppo_acktr import algo
    ps, gs, _ = make()
    opt = algo.AdamW(ps, grads=gs, state_bits=bits, seed=5, max_grad_norm=0.5, **HP)
    opt.step(), opt.step()
    torch.save(opt.state_dict(), tmp_path / 'opt.pt')
    qs = [p.clone() for p in ps]
    other = algo.AdamW(qs, grads=gs, state_bits=bits, lr=1.0)
    other.load_state_dict(torch.load(tmp_path / 'opt.pt', weights_only=True))
    opt.step(), other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and other.steps_done() == 3
    with pytest.raises(ValueError):
        algo.AdamW(ps, grads=gs, state_bits=40 - bits, lr=1.0).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        algo.AdamW(ps[:3], grads=gs[:3], state_bits=bits, lr=1.0).load_state_dict(opt.state_dict())


@pytest.mark.parametrize('bits', [32, 8])
def test_state_before_the_first_step(bits):
    """an optimiser is saved, looked into and restored before there is any gradient"""
    from a2c_ppo_acktr import algo
    ps = [rnd(1, 300).requires_grad_(), rnd(2, 5, 7).requires_grad_()]
    opt = algo.AdamW(ps, state_bits=bits, seed=3, **HP)
    assert opt.offsets() == [0, 512] and not any(t.any() for t in opt.moments())
    sd = opt.state_dict()
    assert sd['step'] == 0
    qs = [p.detach().clone().requires_grad_() for p in ps]
    other = algo.AdamW(qs, state_bits=bits, lr=1.0)
    other.load_state_dict(sd)
    with pytest.raises(RuntimeError, match='no gradient'):
        opt.step()
    for k, (p, q) in enumerate(zip(ps, qs)):
        p.grad, q.grad = rnd(10 + k, *p.shape), rnd(10 + k, *p.shape)
    opt.step(), other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('clip', [None, 0.5])
def test_captured_and_replayed(bits, clip):
    from a2c_ppo_acktr import algo, ops
    runs = []
    for captured in (False, True):
        ps, gs, cs = make(cdt=BF)
        opt = algo.AdamW(ps, grads=gs, copies=cs, state_bits=bits, max_grad_norm=clip, seed=9, **HP)
        opt.step()
        if captured:
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with ops.graph_capture(g):
                opt.step()
        for k in range(4):
            for i, t in enumerate(gs):
                t.copy_(rnd(300 + 20 * k + i, *t.shape, scale=0.1))
            g.replay() if captured else opt.step()
            torch.cuda.synchronize()
        runs.append([p.clone() for p in ps] + [c.clone() for c in cs if c is not None])
        assert opt.steps_done() == 5
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('shapes', [SHAPES, [(1500, 1501)]])
def test_a_clip_norm_that_comes_or_goes_between_replays(bits, shapes):
    """the captured step and eager steps agree whatever the clip norm was at the capture; few and many chunks"""
    from a2c_ppo_acktr import algo, ops
    for first in (None, 0.5):
        runs = []
        for captured in (False, True):
            ps, gs, cs = make(shapes, cdt=BF)
            opt = algo.AdamW(ps, grads=gs, copies=cs, state_bits=bits, max_grad_norm=first, seed=9, **HP)
            opt.step()
            if captured:
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with ops.graph_capture(g):
                    opt.step()
            for clip in (first, 0.25 if first is None else None, 0.125, None, 0.5):
                opt.param_groups[0]['max_grad_norm'] = clip
                if captured:
                    opt.prepare()
                    g.replay()
                else:
                    opt.step()
                torch.cuda.synchronize()
                runs.append([p.clone() for p in ps] + [c.clone() for c in cs if c is not None])
            assert opt.steps_done() == 6
        for k in range(5):
            assert all(torch.equal(a, b) for a, b in zip(runs[k], runs[5 + k])), (first, k)


def test_a_captured_step_follows_the_table():
    """gradients that were replaced by an eager step are what a step captured before reads afterwards; nothing points to freed memory"""
    from a2c_ppo_acktr import algo, ops
    p = rnd(1, 500).requires_grad_()
    p.grad = rnd(2, 500)
    opt = algo.AdamW([p.detach()], grads=None, copies=[None], **HP)
    opt.params[0].grad = p.grad
    opt.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with ops.graph_capture(g):
        opt.step()
    opt.params[0].grad = rnd(3, 500)                         # another tensor
    opt.step()
    want = algo.AdamW([p.detach().clone()], grads=[opt.params[0].grad.clone()], **HP)
    want.load_state_dict(opt.state_dict())
    g.replay()
    want.step()
    assert torch.equal(want.params[0], opt.params[0]) and opt.steps_done() == 3


def test_another_layout_at_the_same_address_is_refused():
    from a2c_ppo_acktr import algo
    p, g = rnd(1, 40, 40), rnd(2, 40, 40)
    opt = algo.AdamW([p], **HP)
    p.grad = g
    opt.step()
    before = p.clone()
    p.grad = g.t()                                           # same memory, size and type
    with pytest.raises(RuntimeError, match='contiguous'):
        opt.step()
    p.grad = g
    opt.step()
    assert opt.steps_done() == 2 and not torch.equal(p, before)


def test_a_tensor_of_more_than_2_31_elements():
    """the last elements of a long tensor take the step that they would take in a short one"""
    from a2c_ppo_acktr import algo
    n, tail = (1 << 31) + 4099, 5000
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    p[-tail:] = rnd(1, tail).bfloat16()
    g[-tail:] = rnd(2, tail).bfloat16()
    q, h = p[-tail:].clone(), g[-tail:].clone()
    long, short = algo.AdamW([p], grads=[g], **HP), algo.AdamW([q], grads=[h], **HP)
    for _ in range(2):
        long.step()
        short.step()
    assert torch.equal(p[-tail:], q) and not p[:4096].any()


def test_refusals():
    from a2c_ppo_acktr import algo
    p, g = rnd(1, 100), rnd(2, 100)
    for f in (lambda: algo.AdamW([], lr=1.0), lambda: algo.AdamW([p], lr=1.0, state_bits=16), lambda: algo.AdamW([p], lr=1.0, grads=[]),
              lambda: algo.AdamW([p], lr=-1.0), lambda: algo.AdamW([p], lr=1.0, betas=(1.0, 0.9)), lambda: algo.AdamW([p], lr=1.0, max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            f()
    for ps, gs, cs in (([p], [rnd(1, 99)], None), ([p], [g.double()], None), ([p, p], [g, g], None), ([p[::2]], [g[::2]], None),
                       ([p], [g.cpu()], None), ([p.cpu()], [g], None), ([p], [g], [p]), ([p, p[50:]], [g, g[50:]], None)):
        with pytest.raises(RuntimeError):
            algo.AdamW(ps, grads=gs, copies=cs, lr=1.0).step()
