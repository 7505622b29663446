"""gated_scan_fwd / _bwd / _step against a step-by-step 64-bit evaluation (gated_refs.py derives the tolerances)."""
import pytest
import torch

from gated_refs import check, scan64

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def inputs(T, N, H, dt, layout='packed', seed=0, shift=1.0):
    if layout == 'packed':                                  # halves of one projection
        proj = (rnd(seed, T, N, 2 * H, scale=2.0) + torch.cat((torch.full((H,), shift), torch.zeros(H))).to(DEV)).to(dt)
        g, v = proj[..., :H], proj[..., H:]
    elif layout == 'batch':                                 # [N, T, H] storage
        g, v = (rnd(seed + i, N, T, H, scale=2.0, dtype=dt).transpose(0, 1) for i in (0, 1))
    else:                                                   # rows of odd pitch
        g, v = (rnd(seed + i, T, N, H + 3, scale=2.0, dtype=dt)[..., :H] for i in (0, 1))
    m = (rnd(seed + 2, T, N) < 1.3).float()                 # a tenth of the steps restart
    return g, v, m, rnd(seed + 3, N, H), rnd(seed + 4, T, N, H, dtype=dt), rnd(seed + 5, N, H)


def run(T, N, H, dt, layout='packed', masked=True, state=True, last=True, seed=0, shift=1.0):
    from a2c_ppo_acktr import ops
    g, v, m, h0, dout, dl = inputs(T, N, H, dt, layout, seed, shift)
    m, h0, dl = m if masked else None, h0 if state else None, dl if last else None
    out, fin, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    dg, dv, dh0 = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)
    ref = scan64(g, v, h0, m, dout, dl)
    for name, t in (('out', out), ('last', fin), ('dgate', dg), ('dvalue', dv), ('dh0', dh0)):
        check(t, ref[name], name)
    o2, f2, none = ops.gated_scan_fwd(g, v, h0, m)
    assert none is None and torch.equal(o2, out) and torch.equal(f2, fin)
    again = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)
    assert all(torch.equal(p, q) for p, q in zip(again, (dg, dv, dh0)))


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('T', [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 128, 129, 255, 256, 257, 513, 1000])
def test_lengths(T, dt):
    run(T, 3, 40, dt)


@pytest.mark.parametrize('dt', [BF, F32])
@pytest.mark.parametrize('N,H', [(1, 1), (1, 3), (2, 4), (5, 63), (4, 64), (3, 65), (1, 1000), (33, 77), (7, 512)])
@pytest.mark.parametrize('T', [5, 130])
def test_widths(N, H, T, dt):
    run(T, N, H, dt)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('layout', ['packed', 'batch', 'odd'])
def test_layouts(dt, layout):
    run(70, 5, 48, dt, layout)
    run(300, 2, 24, dt, layout, seed=9)


@pytest.mark.parametrize('masked,state,last', [(False, True, True), (True, False, True), (True, True, False), (False, False, False)])
def test_optional_operands(masked, state, last):
    run(150, 3, 32, F32, masked=masked, state=state, last=last)
    run(20, 3, 32, BF, masked=masked, state=state, last=last)


@pytest.mark.parametrize('dt', [BF, F32])
@pytest.mark.parametrize('T,N,H', [(3000, 1, 24), (2500, 2, 37), (5000, 1, 8), (700, 64, 256)])
def test_time_is_split_over_workgroups(T, N, H, dt):
    run(T, N, H, dt, shift=4.0)                             # slow gates: states reach across the blocks
    run(T, N, H, dt, masked=False, seed=3, shift=6.0)


@pytest.mark.parametrize('T,N,H,dt', [
    (300, 32, 1024, BF),                 # two channels a lane, 8 waves, whole tiles: three superchunks
    (150, 36, 974, BF), (150, 36, 974, HF),          # the same with tiles of several sequences
    (200, 64, 1024, BF), (333, 64, 1024, HF),        # 4 waves, whole tiles: several superchunks of 64 steps
    (150, 70, 974, BF), (150, 70, 974, HF),          # 4 waves, tiles of several sequences
    (150, 40, 973, BF), (150, 40, 973, F32), (300, 33, 1024, F32),       # one channel a lane, 4 waves
    (8200, 1, 512, BF), (8200, 1, 512, HF),          # two channels a lane, time split over workgroups, whole tiles
    (4500, 5, 190, BF), (4500, 5, 190, HF),          # the same with tiles of several sequences
    (2100, 3, 77, F32), (2100, 3, 77, HF),           # one channel a lane, split, tiles of several sequences
    (16, 64, 1024, BF), (16, 64, 1024, HF), (10, 70, 974, BF), (10, 70, 974, HF),        # two channels a lane, a wave
    (50, 2, 64, BF), (50, 2, 64, HF), (12, 2, 64, BF), (12, 2, 64, HF),                  # one channel a lane, whole tiles, 4 waves and one
])
def test_every_plan(T, N, H, dt):
    run(T, N, H, dt, shift=2.0)


@pytest.mark.parametrize('T,N,H', [(300, 32, 1024), (8200, 1, 512)])
def test_the_two_passes_may_be_laid_out_apart(T, N, H):
    """a backward pass whose derivative has odd rows takes one channel a lane, on states that a forward pass with two has saved"""
    from a2c_ppo_acktr import ops
    g, v, m, h0, dout, dl = inputs(T, N, H, BF, shift=2.0)
    odd = torch.empty(T, N, H + 1, dtype=BF, device=DEV)[..., :H].copy_(dout)
    out, fin, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    got = ops.gated_scan_bwd(odd, g, v, h0, m, saved=saved, dlast=dl)
    ref = scan64(g, v, h0, m, dout, dl)
    for name, t in (('out', out), ('last', fin), ('dgate', got[0]), ('dvalue', got[1]), ('dh0', got[2])):
        check(t, ref[name], name)


def test_many_channels():
    run(40, 96, 768, BF)


def test_extreme_gates():
    """gates that are open, shut, or beyond fp32's exponential"""
    from a2c_ppo_acktr import ops
    T, N, H = 90, 2, 16
    g, v, m, h0, dout, dl = inputs(T, N, H, F32)
    g = g.clone()
    g[::3], g[1::5], g[2::7], g[10], g[11] = 30.0, -30.0, 8.0, 200.0, -200.0
    out, fin, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    dg, dv, dh0 = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)
    ref = scan64(g, v, h0, m, dout, dl)
    for name, t in (('out', out), ('last', fin), ('dgate', dg), ('dvalue', dv), ('dh0', dh0)):
        # e^-200 has no fp32 value: gates below -87 are taken as -87, so f is off by e^-87 = 1.7e-38 there; it is multiplied by the state
        # (at most the largest |h0| or |v|: every step is a weighted mean), by m h - v (at most twice that), by the derivative of the
        # step (at most the sum of all |dout| and |dlast| of a channel: nothing grows on its way back), or by two of them
        r, tol = ref[name]
        top = max(float(h0.abs().max()), float(v.abs().max()))
        back = float((dout.abs().sum(0) + dl.abs()).max())
        check(t, (r, tol + 1.7e-38 * max(2 * top, 1.0) * max(back, 1.0)), name)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('T,N,H', [(90, 2, 16), (3000, 1, 8)])
def test_gates_without_bound(T, N, H, dt):
    """infinite gates, and finite ones whose product with log2(e) has no fp32 value: held open (the state stays) or shut"""
    from a2c_ppo_acktr import ops
    g, v, m, h0, dout, dl = inputs(T, N, H, dt)
    g, inf, most = g.clone(), float('inf'), 65504.0 if dt == HF else 3e38
    g[::5, :, 0], g[::7, :, 1], g[::3, :, 2], g[::4, :, 3] = inf, -inf, most, -most
    g[T // 2, :, 4], g[T // 2 + 1, :, 4], g[:, :, 5] = inf, -inf, inf
    out, fin, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    dg, dv, dh0 = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)
    ref = scan64(g, v, h0, m, dout, dl)
    # as in test_extreme_gates: a shut gate is taken as -87, f = 1.7e-38
    top, back = max(float(h0.abs().max()), float(v.abs().max())), float((dout.abs().float().sum(0) + dl.abs()).max())
    for name, t in (('out', out), ('last', fin), ('dgate', dg), ('dvalue', dv), ('dh0', dh0)):
        r, tol = ref[name]
        check(t, (r, tol + 1.7e-38 * max(2 * top, 1.0) * max(back, 1.0)), name)
    state = h0.clone()
    for t in range(12):
        y = ops.gated_scan_step(g[t], v[t], state, m[t])
        check(y, (ref['out'][0][t], ref['out'][1][t] + 1.7e-38 * 2 * top), t)


def test_a_mask_of_zero_cuts_what_is_not_finite():
    from a2c_ppo_acktr import ops
    for T, N, H in ((200, 2, 16), (40, 1, 5), (3000, 1, 8)):
        g, v, m, h0, dout, dl = inputs(T, N, H, F32)
        m = torch.ones_like(m)
        cut = T // 2 + 1
        m[cut] = 0
        want = ops.gated_scan_fwd(g, v, h0, m)
        bad = v.clone()
        bad[cut - 2, 0, 1], bad[cut - 1, 0, 2] = float('nan'), float('inf')
        h1 = h0.clone()
        h1[0, 0] = float('nan')
        out, last, saved = ops.gated_scan_fwd(g, bad, h1, m, save=True)
        assert torch.equal(out[cut:], want[0][cut:]) and torch.equal(last, want[1])
        assert not bool(out[cut - 1].isfinite().all())
        # gradients: what lies behind the cut does not reach over it
        d2 = dout.clone()
        d2[cut + 1, 0, 3] = float('nan')
        _, _, s2 = ops.gated_scan_fwd(g, v, h0, m, save=True)
        ok = ops.gated_scan_bwd(dout, g, v, h0, m, saved=s2, dlast=dl)
        got = ops.gated_scan_bwd(d2, g, v, h0, m, saved=s2, dlast=dl)
        assert torch.equal(got[0][:cut], ok[0][:cut]) and torch.equal(got[2], ok[2]) and bool(got[0][cut + 1].isnan().any())
        got = ops.gated_scan_bwd(dout, g, bad, h1, m, saved=saved, dlast=dl)
        assert torch.equal(got[0][cut:], ok[0][cut:]) and torch.equal(got[1], ok[1])


@pytest.mark.parametrize('dt', [BF, F32])
@pytest.mark.parametrize('T,N,H,shift', [(3000, 1, 8, 0.0), (400, 3, 40, -12.0), (20, 2, 8, -30.0), (700, 64, 256, -1.0)])
def test_what_is_not_finite_stays_until_a_mask(T, N, H, shift, dt):
    """factors over many steps are far below fp32's smallest number; what they multiply is lost only where a mask is 0"""
    from a2c_ppo_acktr import ops
    g, v, m, h0, dout, dl = inputs(T, N, H, dt, shift=shift)
    m = torch.ones_like(m)
    cut = T * 3 // 4
    m[cut, 0] = 0
    nan, at = float('nan'), T // 3
    out, last, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    dg, dv, dh0 = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)
    # a state, a value: every step up to the cut, and no other channel
    h1, v1 = h0.clone(), v.clone()
    h1[0, 0], h1[-1, 3], v1[at, 0, 1] = nan, float('inf'), nan
    o, l, s1 = ops.gated_scan_fwd(g, v1, h1, m, save=True)
    bad = torch.zeros(T, N, H, dtype=torch.bool, device=DEV)
    bad[:cut, 0, 0], bad[at:cut, 0, 1] = True, True
    bad[:cut if N == 1 else T, -1, 3] = True
    assert torch.equal(~o.isfinite(), bad) and torch.equal(o[~bad], out[~bad])
    assert torch.equal(~l.isfinite(), bad[-1]) and torch.equal(l[~bad[-1]], last[~bad[-1]])
    a, b, _ = ops.gated_scan_bwd(dout, g, v1, h1, m, saved=s1, dlast=dl)
    # (a gate's gradient takes the state before its step)
    assert bool(a[1:cut, 0, 0].isnan().all()) and bool(a[at:cut, 0, 1].isnan().all()) and torch.equal(a[cut:, 0], dg[cut:, 0]) and torch.equal(b, dv)
    # a derivative: every step down to the cut
    d1, l1 = dout.clone(), dl.clone()
    d1[at, 0, 2], l1[0, 4] = nan, nan
    a, b, c = ops.gated_scan_bwd(d1, g, v, h0, m, saved=saved, dlast=l1)
    bad = torch.zeros(T, N, H, dtype=torch.bool, device=DEV)
    bad[:at + 1, 0, 2], bad[cut:, 0, 4] = True, True
    assert torch.equal(a.isnan(), bad) and torch.equal(b.isnan(), bad) and torch.equal(c.isnan(), bad[0])
    assert torch.equal(a[~bad], dg[~bad]) and torch.equal(b[~bad], dv[~bad]) and torch.equal(c[~bad[0]], dh0[~bad[0]])


def test_every_step_masked():
    from a2c_ppo_acktr import ops
    g, v, m, h0, dout, dl = inputs(100, 2, 24, F32)
    m.zero_()
    out, last, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    check(out, scan64(g, v, h0, m)['out'], 'out')
    assert not ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)[2].any()


def test_no_steps_or_sequences():
    from a2c_ppo_acktr import ops
    h0, dl = rnd(1, 3, 8), rnd(2, 3, 8)
    e = torch.empty(0, 3, 8, dtype=BF, device=DEV)
    out, last, saved = ops.gated_scan_fwd(e, e, h0, torch.empty(0, 3, device=DEV), save=True)
    assert out.shape == (0, 3, 8) and torch.equal(last, h0) and saved.shape[0] == 0
    assert torch.equal(ops.gated_scan_bwd(e, e, e, h0, None, saved=saved, dlast=dl)[2], dl)
    assert not ops.gated_scan_bwd(e, e, e)[2].any() and not ops.gated_scan_fwd(e, e)[1].any()
    z = torch.empty(5, 0, 8, dtype=BF, device=DEV)
    assert ops.gated_scan_fwd(z, z)[0].shape == (5, 0, 8)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('N,H', [(1, 1), (32, 512), (3, 77), (7, 6)])
def test_one_step(dt, N, H):
    """the one-token form, driven for several steps, is the sequence form"""
    from a2c_ppo_acktr import ops
    T = 6
    g, v, m, h0, _, _ = inputs(T, N, H, dt)
    ref = scan64(g, v, h0, m)
    state = h0.clone()
    for t in range(T):
        out = ops.gated_scan_step(g[t], v[t], state, m[t] if t % 2 else m[t][:, None])
        check(out, (ref['out'][0][t], ref['out'][1][t]), t)
    check(state, ref['last'], 'state')
    s2 = h0.clone()
    ops.gated_scan_step(g[0], v[0], s2)                     # without masks
    check(s2, scan64(g[:1], v[:1], h0, None)['last'], 'state')


def test_gradients_into_one_projection():
    from a2c_ppo_acktr import ops
    T, N, H = 90, 3, 24
    g, v, m, h0, dout, dl = inputs(T, N, H, BF)
    _, _, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    want = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)
    d = torch.full((T, N, 2 * H + 8), 3.0, dtype=BF, device=DEV)
    ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl, dgate=d[..., :H], dvalue=d[..., H:2 * H])
    assert torch.equal(d[..., :H], want[0]) and torch.equal(d[..., H:2 * H], want[1]) and bool((d[..., 2 * H:] == 3).all())


def test_gradient_against_differences():
    from a2c_ppo_acktr import ops
    T, N, H = 70, 2, 9
    g, v, m, h0, dout, dl = inputs(T, N, H, F32)
    _, _, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    grads = ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dlast=dl)

    def loss(g, v, h):
        h = h.clone()
        total = 0.0
        for t in range(T):
            f = torch.sigmoid(g[t])
            h = f * (m[t][:, None].double() * h) + (1 - f) * v[t]
            total += float((h * dout[t].double()).sum())
        return total + float((h * dl.double()).sum())
    args = [g.double(), v.double(), h0.double()]
    for i in range(3):
        d = rnd(50 + i, *args[i].shape).double()
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + 1e-4 * d, args[i] - 1e-4 * d
        num, ana = (loss(*up) - loss(*dn)) / 2e-4, float((grads[i].double() * d).sum())
        # third derivatives of a step are below 1: the difference is off by 1e-8 / 6 of the gradient's scale, fp32 by 1e-5
        assert abs(num - ana) <= 2e-5 * float(grads[i].double().norm() * d.norm()), (i, num, ana)


@pytest.mark.parametrize('dt', [BF, F32])
@pytest.mark.parametrize('far', ['steps', 'sequences'])
def test_strides_that_need_64_bits(far, dt):
    """a few short rows, gigabytes apart"""
    from a2c_ppo_acktr import ops
    T, N, H = 20, 3, 40
    e = torch.empty(0, dtype=dt).element_size()

    def spread(t):
        if far == 'steps':                                   # 16 steps reach over 2^31 bytes
            return torch.empty(T, (1 << 27) // e + 8, dtype=dt, device=DEV)[:, :N * H].view(T, N, H).copy_(t)
        return torch.empty(N, (1 << 30) // e + 8, dtype=dt, device=DEV)[:, :T * H].view(N, T, H).transpose(0, 1).copy_(t)
    g, v, m, h0, dout, dl = inputs(T, N, H, dt)
    out, dg, dv = spread(torch.zeros_like(dout)), spread(torch.zeros_like(dout)), spread(torch.zeros_like(dout))
    gs, vs, ds = spread(g), spread(v), spread(dout)
    _, fin, saved = ops.gated_scan_fwd(gs, vs, h0, m, out=out, save=True)
    _, _, dh0 = ops.gated_scan_bwd(ds, gs, vs, h0, m, saved=saved, dlast=dl, dgate=dg, dvalue=dv)
    ref = scan64(g, v, h0, m, dout, dl)
    for name, t in (('out', out), ('last', fin), ('dgate', dg), ('dvalue', dv), ('dh0', dh0)):
        check(t, ref[name], name)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('T', [9, 50, 130, 400])
def test_sequences_gigabytes_apart(T, dt):
    """64-bit offsets with a wave, with 4, with 8, and with the time split"""
    from a2c_ppo_acktr import ops
    N, H = 3, 40
    e = torch.empty(0, dtype=dt).element_size()
    spread = lambda t: torch.empty(N, (1 << 30) // e + 8, dtype=dt, device=DEV)[:, :T * H].view(N, T, H).transpose(0, 1).copy_(t)
    g, v, m, h0, dout, dl = inputs(T, N, H, dt)
    gs, vs, ds = spread(g), spread(v), spread(dout)
    out, dg, dv = (spread(torch.zeros_like(dout)) for _ in range(3))
    _, fin, saved = ops.gated_scan_fwd(gs, vs, h0, m, out=out, save=True)
    _, _, dh0 = ops.gated_scan_bwd(ds, gs, vs, h0, m, saved=saved, dlast=dl, dgate=dg, dvalue=dv)
    ref = scan64(g, v, h0, m, dout, dl)
    for name, t in (('out', out), ('last', fin), ('dgate', dg), ('dvalue', dv), ('dh0', dh0)):
        check(t, ref[name], name)


def test_more_than_2_31_elements():
    """a sequence whose last steps lie past 2^31 elements: a restart cuts off what would need a reference of a million steps"""
    from a2c_ppo_acktr import ops
    T, N, H, tail = (1 << 20) + 300, 1, 2048, 200
    g, v = torch.zeros(T, N, H, dtype=BF, device=DEV), torch.zeros(T, N, H, dtype=BF, device=DEV)
    dout, m = torch.zeros(T, N, H, dtype=BF, device=DEV), torch.ones(T, N, device=DEV)
    m[T - tail] = 0
    for i, t in enumerate((g, v, dout)):
        t[-tail:] = rnd(i, tail, N, H, dtype=BF)
    out, fin, saved = ops.gated_scan_fwd(g, v, None, m, save=True)
    dg, dv, dh0 = ops.gated_scan_bwd(dout, g, v, None, m, saved=saved)
    ref = scan64(g[-tail:], v[-tail:], None, m[-tail:], dout[-tail:], None)
    for name, t in (('out', out), ('last', fin), ('dgate', dg), ('dvalue', dv)):
        check(t if name == 'last' else t[-tail:], ref[name], name)
    assert not out[:-tail].any() and not dg[:-tail].any() and not dh0.any()


def test_captured_and_replayed():
    from a2c_ppo_acktr import ops
    for T, N, H in ((150, 4, 64), (4000, 1, 16)):
        g, v, m, h0, dout, dl = inputs(T, N, H, BF)
        base = g._base
        step = lambda: (lambda o: (o[0], o[1]) + ops.gated_scan_bwd(dout, g, v, h0, m, saved=o[2], dlast=dl))(
            ops.gated_scan_fwd(g, v, h0, m, save=True))
        step()
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with ops.graph_capture(gr):
                out = step()
            graphs.append((gr, out))
        for k in range(4):
            base.copy_(rnd(60 + k, *base.shape, dtype=BF))
            want = [t.clone() for t in step()]
            for gr, out in graphs:
                gr.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_refusals_on_the_device():
    from a2c_ppo_acktr import ops
    g, v, m, h0, dout, dl = inputs(100, 2, 8, BF)
    _, _, saved = ops.gated_scan_fwd(g, v, h0, m, save=True)
    bad = [lambda: ops.gated_scan_fwd(g, v.float(), h0, m), lambda: ops.gated_scan_fwd(g, v[:50], h0, m),
           lambda: ops.gated_scan_fwd(g, v, h0.bfloat16(), m), lambda: ops.gated_scan_fwd(g, v, h0[:1], m),
           lambda: ops.gated_scan_fwd(g, v, h0, m[:50]), lambda: ops.gated_scan_fwd(g, v, h0, m.bool()),
           lambda: ops.gated_scan_fwd(g, v, h0, m, out=g), lambda: ops.gated_scan_fwd(g, v, h0, m, out=dout[:1].expand(100, 2, 8)),
           lambda: ops.gated_scan_fwd(g.transpose(1, 2), v.transpose(1, 2)),
           lambda: ops.gated_scan_bwd(dout, g, v, h0, m), lambda: ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved[:1]),
           lambda: ops.gated_scan_bwd(dout[:, :1], g, v, h0, m, saved=saved),
           lambda: ops.gated_scan_bwd(dout, g, v, h0, m, saved=saved, dgate=dout),
           lambda: ops.gated_scan_step(g[0], v[0], h0.bfloat16()), lambda: ops.gated_scan_step(g[0], v[0], h0.t().contiguous().t()),
           lambda: ops.gated_scan_step(g[0], v[0], h0, m[0][:1])]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()


def test_a_shared_row_in_the_state_is_refused():
    """a gate or value row that all sequences share may not reach into the state that the step updates"""
    from a2c_ppo_acktr import ops
    N, H = 4, 16
    buf = rnd(1, N * H + 3 * H)
    row, other, state = buf[:H].expand(N, H), buf[-H:].expand(N, H), buf[H // 2:H // 2 + N * H].view(N, H)
    for g, v in ((row, other), (other, row)):
        with pytest.raises(RuntimeError, match='overlaps'):
            ops.gated_scan_step(g, v, state)
    state = buf[H:H + N * H].view(N, H)                      # apart from both rows
    want = scan64(row[None], other[None], state.clone(), None)['out']
    check(ops.gated_scan_step(row, other, state), (want[0][0], want[1][0]), 'out')
