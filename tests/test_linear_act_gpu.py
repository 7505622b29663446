"""linear_act_fwd / linear_act_bwd against a 64-bit evaluation (gated_refs.py derives the tolerances)."""
import pytest
import torch

from gated_refs import ACTS, check, linear64, linear_grads64
from gated_refs import E32, EPS, TINY, act64

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def run(M, N, K, dt, act, bias=True, res=True, pad=0, seed=0, big=1.0):
    from a2c_ppo_acktr import ops
    cut = lambda s, r, c, k=1.0: rnd(seed + s, r, c + pad, scale=k, dtype=dt)[:, :c]
    x, w = cut(1, M, K, big), cut(2, N, K, 1.5 / K ** 0.5)
    b = rnd(seed + 3, N, scale=0.5, dtype=dt) if bias else None
    r = cut(4, M, N) if res else None
    dy = cut(5, M, N, 0.1)
    pre = torch.empty(M, N, dtype=dt, device=DEV) if act != 'none' else None
    y = ops.linear_act_fwd(x, w, b, act=act, residual=r, pre=pre)
    dx, dw, db = ops.linear_act_bwd(dy, x, w, pre=pre, act=act)
    ry, ty, slope, ts = linear64(x, w, b, act, r)
    gx, gw, gb = linear_grads64(dy, x, w, slope, ts)
    check(y, (ry, ty), 'y')
    check(dx, gx, 'dx')
    check(dw, gw, 'dw')
    check(db, gb, 'db')
    # without pre the same values come out
    assert torch.equal(ops.linear_act_fwd(x, w, b, act=act, residual=r), y)
    # and again, bit for bit
    again = ops.linear_act_bwd(dy, x, w, pre=pre, act=act)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


SIZES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 64, 64), (16, 16, 32), (17, 33, 65), (32, 1024, 512), (33, 40, 200), (64, 64, 64), (65, 129, 8),
         (128, 256, 72), (130, 264, 136), (255, 257, 96), (300, 96, 1000), (1011, 390, 777), (512, 512, 512), (1000, 16, 2048)]


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('M,N,K', SIZES)
def test_sizes(M, N, K, dt):
    run(M, N, K, dt, 'tanh')


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('bias,res', [(False, False), (True, False), (False, True)])
def test_epilogues(act, dt, bias, res):
    run(200, 136, 96, dt, act, bias, res)
    run(70, 37, 51, dt, act, bias, res, seed=50)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('pad', [1, 3, 4, 8, 40])
def test_rows_of_wider_tensors(dt, pad):
    run(140, 72, 104, dt, 'silu', pad=pad)


@pytest.mark.parametrize('dt', [BF, F32])
@pytest.mark.parametrize('M,N,K', [(4096, 512, 1568), (2048, 1024, 512), (8200, 260, 136), (16, 2048, 2048), (5000, 8, 40), (20000, 24, 16)])
def test_larger(dt, M, N, K):
    run(M, N, K, dt, 'gelu')


@pytest.mark.parametrize('dt', [BF, HF])
@pytest.mark.parametrize('M,N,K', [(8190, 4090, 264), (8190, 136, 4088), (300, 4088, 4090), (8192, 4096, 128)])
def test_largest_tiles_with_ragged_edges(dt, M, N, K):
    """forward, input gradient and weight gradient, in turn, fill two or one rounds of 256 x 256 tiles, with cut edges"""
    run(M, N, K, dt, 'silu')


# One shape, with ragged edges, for every kernel that the estimate in linear_act.hpp can pick: product, tile, split reduction or not.
TILES16 = [
    ('forward', 84, 70, 913),            # 64 x 64, split
    ('forward', 8249, 72, 74),           # 128 x 64
    ('forward', 1426, 73, 1473),         # 128 x 64, split
    ('forward', 16647, 324, 72),         # 128 x 128
    ('forward', 4090, 2046, 520),        # 128 x 128
    ('forward', 5453, 72, 3920),         # 128 x 128, split
    ('forward', 19769, 520, 76),         # 256 x 256
    ('forward', 16605, 193, 3652),       # 256 x 256, split
    ('dx', 73, 73, 71),                  # 64 x 64
    ('dx', 73, 897, 70),                 # 64 x 64, split
    ('dx', 8249, 72, 74),                # 128 x 64
    ('dx', 76, 3278, 595),               # 128 x 64, split
    ('dx', 14063, 72, 401),              # 128 x 128
    ('dx', 5620, 3912, 72),              # 128 x 128, split
    ('dx', 19598, 72, 555),              # 256 x 256
    ('dx', 17391, 3920, 196),            # 256 x 256, split
    ('dw', 73, 73, 71),                  # 64 x 64
    ('dw', 903, 71, 75),                 # 64 x 64, split
    ('dw', 71, 195, 4139),               # 128 x 64
    ('dw', 7152, 71, 280),               # 128 x 64, split
    ('dw', 71, 1440, 4240),              # 128 x 128
    ('dw', 11909, 1828, 71),             # 128 x 128, split
    ('dw', 300, 4088, 4090),             # 256 x 256
    ('dw', 10758, 137, 4242),            # 256 x 256, split
    ('both', 73, 73, 71),                # one launch, dx in 64 x 64
    ('both', 903, 71, 75),               # one launch, dx in 64 x 64, dw split
    ('both', 201, 132, 4286),            # one launch, dx in 128 x 64
    ('both', 7134, 77, 215),             # one launch, dx in 128 x 64, dw split
    ('both', 16380, 2044, 2050),         # apart: dx in 128 x 128, dw in 256 x 256, split
]
TILES32 = [
    ('forward', 76, 70, 314), ('forward', 19780, 129, 71), ('forward', 75, 3065, 1413),         # 64 x 64 split; 128 x 64; the same split
    ('dx', 70, 71, 76), ('dx', 73, 290, 74), ('dx', 17770, 73, 130), ('dx', 2870, 1439, 72),    # 64 x 64, split; 128 x 64, split
    ('dw', 70, 71, 76), ('dw', 301, 71, 71), ('dw', 70, 4803, 647), ('dw', 1439, 72, 3006),
    ('both', 70, 71, 76), ('both', 301, 71, 71), ('both', 841, 74, 1293), ('both', 333, 4085, 4309),
]


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('act', ['none', 'gelu'])
@pytest.mark.parametrize('M,N', [(1, 1), (777, 35), (5000, 264)])
def test_bias_gradient_alone(M, N, act, dt):
    from a2c_ppo_acktr import ops
    x, w, dy = rnd(1, M, 24, dtype=dt), rnd(2, N, 24, scale=0.3, dtype=dt), rnd(3, M, N, dtype=dt)
    pre = torch.empty(M, N, dtype=dt, device=DEV) if act != 'none' else None
    ops.linear_act_fwd(x, w, act=act, pre=pre)
    dx, dw, db = ops.linear_act_bwd(dy, x, w, pre=pre, act=act, need_dx=False, need_dw=False)
    _, _, slope, ts = linear64(x, w, None, act)
    assert dx is None and dw is None
    check(db, linear_grads64(dy, x, w, slope, ts)[2], 'db')


@pytest.mark.parametrize('dt,what,M,N,K', [(dt,) + t for dt in (BF, HF) for t in TILES16] + [(F32,) + t for t in TILES32])
def test_every_kernel(dt, what, M, N, K):
    from a2c_ppo_acktr import ops
    x, w = rnd(1, M, K, dtype=dt), rnd(2, N, K, scale=1.5 / K ** 0.5, dtype=dt)
    b, r, dy = rnd(3, N, scale=0.5, dtype=dt), rnd(4, M, N, dtype=dt), rnd(5, M, N, scale=0.1, dtype=dt)
    pre = torch.empty(M, N, dtype=dt, device=DEV)
    y = ops.linear_act_fwd(x, w, b, act='silu', residual=r, pre=pre)
    ry, ty, slope, ts = linear64(x, w, b, 'silu', r)
    check(y, (ry, ty), 'y')
    if what == 'forward':
        assert all(torch.equal(ops.linear_act_fwd(x, w, b, act='silu', residual=r), y) for _ in range(3))
        return
    need = dict(need_dx=what != 'dw', need_dw=what != 'dx', need_db=what != 'dx')
    got = ops.linear_act_bwd(dy, x, w, pre=pre, act='silu', **need)
    for name, t, ref in zip(('dx', 'dw', 'db'), got, linear_grads64(dy, x, w, slope, ts)):
        if t is not None:
            check(t, ref, name)
    for _ in range(3):
        again = ops.linear_act_bwd(dy, x, w, pre=pre, act='silu', **need)
        assert all(p is None if q is None else torch.equal(p, q) for p, q in zip(again, got))


def test_large_pre_activations():
    """tails of every activation: values far from zero"""
    for act in ACTS:
        run(96, 64, 64, F32, act, big=30.0)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('act', ['tanh', 'silu', 'gelu'])
def test_tails_are_right_relative_to_their_own_size(act, dt):
    """Values and slopes of negative pre-activations, which an identity weight makes exact, down to where the exponential is 0.
    With E = 2^-24: the exponential is off by 4 E (exp2 2, its correction 1), 1 + e by 1, a reciprocal by 2, a product by 1; the
    polynomial of gelu's tail, its argument's reciprocal included, by 8.  silu: 4 + 1 + 2 + 1 + 1, gelu: 4 + 8 + 1 + 1: 16 E.  tanh goes
    through 1 - e, which is 0.39 and more where it is used, 4 E 0.61 / 0.39 + 1 + 3 + 1 = 12, or a series (its next term 3.3e-7 = 6 E, its
    roundings 4).  16-bit storage does not carry the rounding of the exponent, E z^2 for gelu (two of z^2 / 2), E |z| for silu, 2 E |z| for tanh."""
    from a2c_ppo_acktr import ops
    low = {'tanh': 40.0, 'silu': 86.0, 'gelu': 12.8}[act]
    x = torch.cat((torch.linspace(-low, 0.0, 40000, device=DEV), torch.linspace(0.0, 6.0, 4000, device=DEV))).to(dt).view(-1, 8)
    pre = torch.empty_like(x)
    y = ops.linear_act_fwd(x, torch.eye(8, dtype=dt, device=DEV), act=act, pre=pre)
    z = x.double()
    ref, slope = act64(z, act)
    rel = 16 * E32 + (0 if dt == F32 else E32 * {'tanh': 2 * z.abs(), 'silu': z.abs(), 'gelu': z * z}[act])
    check(y, (ref, (rel * (1 + EPS[dt]) + (EPS[dt] if dt != F32 else 0)) * ref.abs() + TINY[dt] + 2.0 ** -118), 'y')
    if dt == F32:                                            # (16 bits: fixed-point steps)
        # tanh 4 e r^2: 4 + 2 (1 + 2) + 3.  silu s (1 + z ns) and gelu Q - a phi have a root at -1.28 and at -0.75; from -2 down their two terms
        # are at most 2.4 and 1.6 times the result: 8 + 2.4 (4 + 1) + 2 and 1.6 (13 + 1) + 1.  Elsewhere to the same part of 1.13.
        d, big = (pre.double() - slope).abs(), 24 * E32
        tol = torch.where((z <= -2) | (act == 'tanh'), slope.abs(), torch.full_like(z, 1.13)) * big + 2.0 ** -118
        assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize('dt', [BF, HF, F32])
def test_activations_at_infinity(dt):
    """limits of values and gradients where the definition has them: act(+inf) = inf, slope 1 (tanh: 1, 0); relu and tanh at -inf"""
    from a2c_ppo_acktr import ops
    inf = float('inf')
    x, w = torch.tensor([[inf], [-inf], [0.5]], dtype=dt, device=DEV), torch.ones(1, 1, dtype=dt, device=DEV)
    for act, top, low in (('relu', inf, 0.0), ('tanh', 1.0, -1.0), ('silu', inf, None), ('gelu', inf, None)):
        pre = torch.empty(3, 1, dtype=dt, device=DEV)
        y = ops.linear_act_fwd(x, w, act=act, pre=pre)
        assert float(y[0]) == top and (low is None or float(y[1]) == low), act
        if act in ('relu', 'tanh', 'gelu'):
            dx, _, _ = ops.linear_act_bwd(torch.ones(3, 1, dtype=dt, device=DEV), x, w, pre=pre, act=act, need_dw=False, need_db=False)
            assert float(dx[0]) == (0.0 if act == 'tanh' else 1.0) and float(dx[1]) == 0.0, act


def test_slices_at_odd_offsets():
    """operands that start in the middle of 16 bytes"""
    from a2c_ppo_acktr import ops
    for off in (1, 2, 5):
        x = rnd(1, 50 * 64 + 16, dtype=BF)[off:off + 50 * 64].view(50, 64)
        w = rnd(2, 24 * 64 + 16, scale=0.1, dtype=BF)[off:off + 24 * 64].view(24, 64)
        out = torch.full((50 * 24 + 16,), 7.0, dtype=BF, device=DEV)
        o = out[off:off + 50 * 24].view(50, 24)
        assert ops.linear_act_fwd(x, w, act='relu', out=o).data_ptr() == o.data_ptr()
        y, t, _, _ = linear64(x, w, None, 'relu')
        check(o, (y, t), 'y')
        assert bool((out[:off] == 7).all()) and bool((out[off + 50 * 24:] == 7).all())      # nothing beside it


def test_rows_beside_the_output_stay():
    from a2c_ppo_acktr import ops
    for M, N, ld in ((70, 37, 64), (130, 64, 80), (5, 24, 25)):
        big = torch.full((M + 3, ld), 5.0, dtype=BF, device=DEV)
        ops.linear_act_fwd(rnd(1, M, 40, dtype=BF), rnd(2, N, 40, dtype=BF), out=big[:M, :N])
        assert bool((big[M:] == 5).all()) and bool((big[:, N:] == 5).all())


def test_no_rows():
    from a2c_ppo_acktr import ops
    x, w = torch.empty(0, 24, dtype=BF, device=DEV), rnd(1, 16, 24, dtype=BF)
    assert ops.linear_act_fwd(x, w, act='gelu').shape == (0, 16)
    pre, dy = torch.empty(0, 16, dtype=BF, device=DEV), torch.empty(0, 16, dtype=BF, device=DEV)
    dx, dw, db = ops.linear_act_bwd(dy, x, w, pre=pre, act='gelu')
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


def test_residual_in_place():
    from a2c_ppo_acktr import ops
    for M, N, K in ((64, 64, 64), (513, 200, 96), (40, 8, 2048)):
        x, w, r = rnd(1, M, K, dtype=BF), rnd(2, N, K, scale=0.1, dtype=BF), rnd(3, M, N, dtype=BF)
        want = ops.linear_act_fwd(x, w, act='silu', residual=r)
        assert torch.equal(ops.linear_act_fwd(x, w, act='silu', residual=r, out=r), want)


@pytest.mark.parametrize('dt', [BF, HF, F32])
@pytest.mark.parametrize('M,N,K', [(70, 37, 51), (200, 136, 96), (4096, 64, 512)])
def test_addend_of_the_input_gradient(dt, M, N, K):
    """dx = dz w + dx_add is rounded once: an addend of the product's size costs one fp32 rounding more; in place too"""
    from a2c_ppo_acktr import ops
    from gated_refs import E32, EPS, TINY
    x, w, dy, add = rnd(1, M, K, dtype=dt), rnd(2, N, K, scale=0.1, dtype=dt), rnd(3, M, N, dtype=dt), rnd(4, M, K, dtype=dt)
    _, _, slope, ts = linear64(x, w)
    (r, t), _, _ = linear_grads64(dy, x, w, slope, ts)
    total = r + add.double()
    t = t - EPS[dt] * r.abs() + (EPS[dt] + E32) * total.abs() + E32 * add.double().abs() + TINY[dt]
    for need in (True, False):
        dx, _, _ = ops.linear_act_bwd(dy, x, w, dx_add=add, need_dw=need, need_db=need)
        check(dx, (total, t), 'dx')
    again, _, _ = ops.linear_act_bwd(dy, x, w, dx_add=add, dx=add)
    assert again.data_ptr() == add.data_ptr() and torch.equal(again, dx)


def test_only_what_is_needed():
    from a2c_ppo_acktr import ops
    x, w, dy = rnd(1, 100, 72, dtype=BF), rnd(2, 40, 72, dtype=BF), rnd(3, 100, 40, dtype=BF)
    pre = torch.empty(100, 40, dtype=BF, device=DEV)
    ops.linear_act_fwd(x, w, act='tanh', pre=pre)
    full = ops.linear_act_bwd(dy, x, w, pre=pre, act='tanh')
    for k in range(3):
        need = [i == k for i in range(3)]
        part = ops.linear_act_bwd(dy, x, w, pre=pre, act='tanh', need_dx=need[0], need_dw=need[1], need_db=need[2])
        for i in range(3):
            assert (part[i] is None) if i != k else torch.equal(part[i], full[i])


def test_values_that_are_not_finite_stay_in_their_rows():
    from a2c_ppo_acktr import ops
    x, w = rnd(1, 150, 64, dtype=BF), rnd(2, 72, 64, dtype=BF)
    clean = ops.linear_act_fwd(x, w, act='silu')
    x2 = x.clone()
    x2[7, 3], x2[149, 63] = float('nan'), float('inf')
    got = ops.linear_act_fwd(x2, w, act='silu')
    keep = [i for i in range(150) if i not in (7, 149)]
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[7].isnan().all()) and not bool(got[149].isfinite().all())
    assert bool(ops.linear_act_fwd(x2, w, act='relu')[7].isnan().all())


def test_gradient_against_differences():
    """fp32: (L(p + h) - L(p - h)) / 2h with L in 64 bits, against the operator's gradients along random directions.  The central
    difference is off by h^2 / 6 times the third derivative, here below 1e-5 of the gradient's scale, the operator by 1e-5."""
    from a2c_ppo_acktr import ops
    for act in ('tanh', 'silu', 'gelu'):
        x, w, b, r = rnd(1, 40, 24), rnd(2, 16, 24, scale=0.3), rnd(3, 16), rnd(4, 40, 16)
        dy = rnd(5, 40, 16)
        pre = torch.empty(40, 16, device=DEV)
        ops.linear_act_fwd(x, w, b, act=act, residual=r, pre=pre)
        dx, dw, db = ops.linear_act_bwd(dy, x, w, pre=pre, act=act)
        loss = lambda x, w, b: float((linear64(x, w, b, act)[0] * dy.double()).sum())
        for i, (p, g) in enumerate(((x, dx), (w, dw), (b, db))):
            v = rnd(10 + i, *p.shape).double()
            h = 1e-4
            args = [x.double(), w.double(), b.double()]
            up, dn = list(args), list(args)
            up[i], dn[i] = args[i] + h * v, args[i] - h * v
            num = (loss(*up) - loss(*dn)) / (2 * h)
            ana = float((g.double() * v).sum())
            assert abs(num - ana) <= 2e-5 * float(g.double().norm() * v.norm()), (act, i, num, ana)


def test_captured_and_replayed():
    from a2c_ppo_acktr import ops
    M, N, K = 260, 136, 72
    x, w, b, dy = rnd(1, M, K, dtype=BF), rnd(2, N, K, dtype=BF), rnd(3, N, dtype=BF), rnd(4, M, N, dtype=BF)
    pre = torch.empty(M, N, dtype=BF, device=DEV)

    def step():
        y = ops.linear_act_fwd(x, w, b, act='gelu', pre=pre)
        return (y,) + ops.linear_act_bwd(dy, x, w, pre=pre, act='gelu')
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                     # two graphs, replayed in turn: neither uses the other's scratch
        g = torch.cuda.CUDAGraph()
        with ops.graph_capture(g):
            out = step()
        graphs.append((g, out))
    for k in range(4):
        x.copy_(rnd(20 + k, M, K, dtype=BF))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_more_than_2_31_elements():
    """the last rows of a product whose rows reach past 2^31 elements; gradients that only those rows have"""
    from a2c_ppo_acktr import ops
    M, N, K, tail = (1 << 20) + 700, 2048, 24, 300
    x, w, b = rnd(1, M, K, dtype=BF), rnd(2, N, K, scale=0.3, dtype=BF), rnd(3, N, dtype=BF)
    pre = torch.empty(M, N, dtype=BF, device=DEV)
    y = ops.linear_act_fwd(x, w, b, act='silu', pre=pre)
    dy = torch.zeros(M, N, dtype=BF, device=DEV)
    dy[-tail:] = rnd(4, tail, N, scale=0.1, dtype=BF)
    dx, dw, db = ops.linear_act_bwd(dy, x, w, pre=pre, act='silu')
    ry, ty, slope, ts = linear64(x[-tail:], w, b, 'silu', None)
    gx, gw, gb = linear_grads64(dy[-tail:], x[-tail:], w, slope, ts)
    check(y[-tail:], (ry, ty), 'y')
    check(dx[-tail:], gx, 'dx')
    check(dw, gw, 'dw')
    check(db, gb, 'db')
    assert not dx[:-tail].any()


@pytest.mark.parametrize('act', ['none', 'relu'])
def test_most_rows(act):
    """gradients whose sums over rows end just below 2^31, in blocks and slices whose nominal ends pass 2^31"""
    from a2c_ppo_acktr import ops
    M, N, K, tail = (1 << 31) - 257, 8, 8, 3000
    x, dy = torch.zeros(M, K, dtype=BF, device=DEV), torch.zeros(M, N, dtype=BF, device=DEV)
    x[-tail:], dy[-tail:] = rnd(1, tail, K, dtype=BF), rnd(2, tail, N, dtype=BF)
    x[:tail], dy[:tail] = rnd(3, tail, K, dtype=BF), rnd(4, tail, N, dtype=BF)
    w = rnd(5, N, K, dtype=BF)
    part = lambda t: torch.cat((t[:tail], t[-tail:]))
    pre = slope = None
    if act != 'none':
        pre = torch.empty(M, N, dtype=BF, device=DEV)
        y = ops.linear_act_fwd(x, w, act=act, pre=pre)
        ry, ty, slope, ts = linear64(part(x), w, None, act)
        check(part(y), (ry, ty), 'y')
        del y
    else:
        slope, ts = torch.ones(2 * tail, N, dtype=torch.float64, device=DEV), torch.zeros(2 * tail, N, dtype=torch.float64, device=DEV)
    _, dw, db = ops.linear_act_bwd(dy, x, w, pre=pre, act=act, need_dx=False)
    # rows of zeros add nothing, however many: the tolerance is that of the rows that have values
    _, gw, gb = linear_grads64(part(dy), part(x), w, slope, ts)
    check(dw, gw, 'dw')
    check(db, gb, 'db')


def test_two_streams():
    from a2c_ppo_acktr import ops
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x, w = rnd(1, 900, 777, dtype=BF), rnd(2, 390, 777, dtype=BF)
    x2, w2 = rnd(3, 900, 777, dtype=BF), rnd(4, 390, 777, dtype=BF)
    want, want2 = ops.linear_act_fwd(x, w, act='silu'), ops.linear_act_fwd(x2, w2, act='silu')
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        with torch.cuda.stream(a):
            got.append((ops.linear_act_fwd(x, w, act='silu'), want))
        with torch.cuda.stream(b):
            got.append((ops.linear_act_fwd(x2, w2, act='silu'), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in got)


def test_refusals_on_the_device():
    from a2c_ppo_acktr import ops
    x, w = rnd(1, 8, 16, dtype=BF), rnd(2, 4, 16, dtype=BF)
    bad = [lambda: ops.linear_act_fwd(x, w.half()), lambda: ops.linear_act_fwd(x, w[:, :8]), lambda: ops.linear_act_fwd(x, w, act='elu'),
           lambda: ops.linear_act_fwd(x, w, bias=rnd(3, 5, dtype=BF)), lambda: ops.linear_act_fwd(x, w, residual=rnd(3, 8, 5, dtype=BF)),
           lambda: ops.linear_act_fwd(x.t(), w.t()), lambda: ops.linear_act_fwd(x.double(), w.double()),
           lambda: ops.linear_act_fwd(x, w, out=x[:, :4]), lambda: ops.linear_act_fwd(x, w, out=rnd(3, 1, 4, dtype=BF).expand(8, 4)),
           lambda: ops.linear_act_fwd(x[:1].expand(8, 16), w), lambda: ops.linear_act_bwd(rnd(3, 8, 4, dtype=BF), x, w, act='tanh'),
           lambda: ops.linear_act_bwd(rnd(3, 8, 5, dtype=BF), x, w), lambda: ops.linear_act_bwd(rnd(3, 8, 4, dtype=BF), x, w, dx=x)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
