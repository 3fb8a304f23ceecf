"""Group norm with its activation (mmdgan_gn_fwd / mmdgan_gn_bwd) against the definition in 64 bits.

Tolerances (u = 2^-24, half a step of fp32 relative to the value).  The kernels evaluate everything on an element in 64 bits and
round once, so y is within u of |y|; lrelu adds the rounding of the product with 0.1 and of 0.1 itself (3 u in all); tanh
rounds its argument first and tanhf is good to two steps (8 u).  dx is rounded once: u |dx|, with 1e-13 of the terms it is
a difference of for the 64-bit arithmetic.  tanh's derivative 1 - t^2 inherits 2 |t| times tanhf's error, at most 12 u of 1, and dz is
rounded once more (u): 13 u of each term |rstd gamma dy| (2 + |xhat|), the means being at most the largest term."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = float(np.float32(1e-5))     # eps is a float argument of the entry: 2.5e-13 away from 1e-5, which the statistics show


@pytest.fixture(scope='module')
def ops():
    from mmdgan_hip import ops as o
    o.require_device()
    return o


def act64(z, act):
    return {'linear': z, 'relu': z.clamp(min=0), 'lrelu': torch.where(z > 0, z, 0.1 * z), 'tanh': torch.tanh(z)}[act]


def forward64(x, gamma, beta, G, act, eps=EPS):
    """y, mean, rstd, xhat of [N, HW, C] doubles (CPU)"""
    N, HW, C = x.shape
    v = x.view(N, HW, G, C // G)
    mean = v.mean(dim=(1, 3))
    d = v - mean.view(N, 1, G, 1)
    rstd = 1.0 / torch.sqrt(d.square().mean(dim=(1, 3)) + eps)
    xhat = (d * rstd.view(N, 1, G, 1)).reshape(N, HW, C)
    return act64(xhat * gamma + beta, act), mean, rstd, xhat


def backward64(x, dy, gamma, beta, G, act):
    N, HW, C = x.shape
    _, _, rstd, xhat = forward64(x, gamma, beta, G, 'linear')
    z = xhat * gamma + beta
    slope = {'linear': torch.ones_like(z), 'relu': (z > 0).double(), 'lrelu': torch.where(z > 0, 1.0, 0.1).double(),
             'tanh': 1 - torch.tanh(z) ** 2}[act]
    dz = dy * slope
    t, q = (dz * gamma).view(N, HW, G, -1), xhat.view(N, HW, G, -1)
    r = rstd.view(N, 1, G, 1)
    dx = r * (t - t.mean(dim=(1, 3), keepdim=True) - q * (t * q).mean(dim=(1, 3), keepdim=True))
    terms = (r * (dy * gamma).abs().view(N, HW, G, -1).amax(dim=(1, 3), keepdim=True) * (2 + q.abs())).reshape(N, HW, C)
    return dx.reshape(N, HW, C), (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1)), terms, dz, xhat


def data(N, HW, C, seed, extra=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, HW, C, generator=g) * 1.5 + 3.0 * torch.rand(C, generator=g)).float()
    return (x, (1 + 0.3 * torch.randn(C, generator=g)).float(), (0.3 * torch.randn(C, generator=g)).float(),
            torch.randn(N + extra, HW, C, generator=g).float())


# (N, HW, C, G): the resident form at several slab widths, the two-pass form (ragged channels, groups wider than a slab, images
# beyond a slab's registers), one pixel, one channel, one group, one channel per group, sizes around the thread counts
GEOMETRIES = [(1, 1, 4, 1), (1, 1, 512, 32), (5, 16, 512, 32), (64, 256, 64, 32), (3, 1024, 64, 32), (2, 4096, 64, 16), (2, 4096, 16, 1),
              (300, 4, 64, 64), (2500, 1, 128, 4), (2, 1023, 32, 8), (2, 1025, 32, 8), (3, 65, 48, 12), (1, 16385, 8, 2), (2, 9000, 4, 4),
              (3, 7, 3, 1), (4, 35, 96, 32), (2, 33, 200, 200), (2, 17, 260, 1), (3, 9, 1200, 2), (2, 5, 768, 1), (1, 3, 1031, 1),
              (2, 130, 254, 127), (1, 5000, 6, 3), (1, 1, 1, 1), (2, 600, 1024, 1)]


@pytest.mark.parametrize('N,HW,C,G', GEOMETRIES)
def test_forward_and_backward_match_the_definition(ops, N, HW, C, G):
    for i, act in enumerate(('linear', 'relu', 'lrelu', 'tanh')):
        print(N, HW, C, G, act, flush=True)
        x, gamma, beta, dy = data(N, HW, C, 7 * C + i)
        y, stats = ops.group_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), G, act=act)
        ry, rmean, rrstd, _ = forward64(x.double(), gamma.double(), beta.double(), G, act)
        assert ((y.cpu().double() - ry).abs() <= (1, 1, 3, 8)[i] * U * ry.abs() + 1e-13).all()
        st = stats.cpu()
        # E[x^2] - mean^2 in 64 bits: 2^-53 of (mean^2 + var) per rounding, a few dozen roundings, against var + eps
        assert ((st[:, :, 0] - rmean).abs() <= 1e-12 * (1 + rmean.abs())).all()
        assert ((st[:, :, 1] - rrstd).abs() <= 64 * 2.0 ** -53 * (rmean ** 2 + 10) * rrstd ** 3 + 1e-14 * rrstd).all()
        dx, dgamma, dbeta = ops.group_norm_bwd(x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda(), stats, act=act)
        rx, rg, rb, terms, dz, xhat = backward64(x.double(), dy.double(), gamma.double(), beta.double(), G, act)
        slack = 13 * U if act == 'tanh' else 1e-13
        # (rstd of the kernel's own statistics: their error above, relative)
        rel = (64 * 2.0 ** -53 * (rmean ** 2 + 10) * rrstd ** 2).max().item() * 3
        assert ((dx.cpu().double() - rx).abs() <= U * rx.abs() + (slack + rel) * terms).all()
        a = dy.double().abs()
        assert ((dgamma.cpu().double() - rg).abs() <= U * rg.abs() + (slack + rel) * (a * (xhat.abs() + 1)).sum(dim=(0, 1))).all()
        assert ((dbeta.cpu().double() - rb).abs() <= U * rb.abs() + slack * a.sum(dim=(0, 1))).all()


@pytest.mark.parametrize('N,HW,C,G', [(33, 1457, 96, 32), (5, 100, 48, 16), (3, 77, 20, 4), (2, 600, 160, 32), (300, 9, 60, 12), (1, 16, 252, 4), (2, 333, 192, 32),
                                      (3, 200, 96, 8), (1100, 3, 12, 4), (2, 2900, 12, 4), (1, 1, 12, 4), (2, 40, 240, 4), (2, 700, 252, 4), (1, 5000, 12, 4)])
def test_groups_that_are_no_power_of_two(ops, N, HW, C, G):
    """3, 5, 6, 12, 60, 63 channels a group, from one pixel to more than a workgroup keeps, more images than workgroups"""
    test_forward_and_backward_match_the_definition(ops, N, HW, C, G)


@pytest.mark.parametrize('N,HW,C,G,act', [(3, 40, 32, 8, 'tanh'), (2, 33, 15, 5, 'tanh'), (2, 2100, 64, 2, 'linear')])
def test_gradient_against_differences(ops, N, HW, C, G, act):
    """<dx, v> against the central difference of sum(y dy) along v, in 64 bits: O(h^2) with h = 1e-4 and derivatives of a few
    units, 1e-6 of the sum of absolute values; fp32's rounding of dx is far below that"""
    x, gamma, beta, dy = data(N, HW, C, 3)
    g = torch.Generator().manual_seed(5)
    v = torch.randn(N, HW, C, generator=g).double()
    vg, vb = torch.randn(C, generator=g).double(), torch.randn(C, generator=g).double()
    xd, gd, bd, dyd = x.double(), gamma.double(), beta.double(), dy.double()
    h = 1e-4
    f = lambda s: (forward64(xd + s * h * v, gd + s * h * vg, bd + s * h * vb, G, act)[0] * dyd).sum()
    want = (f(1) - f(-1)) / (2 * h)
    _, stats = ops.group_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), G, act=act)
    dx, dg, db = ops.group_norm_bwd(x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda(), stats, act=act)
    parts = (dx.cpu().double() * v, dg.cpu().double() * vg, db.cpu().double() * vb)
    got = sum(p.sum() for p in parts)
    assert abs(got - want) <= 1e-6 * sum(p.abs().sum() for p in parts)


@pytest.mark.parametrize('HW,C,G', [(64, 32, 8), (37, 15, 5), (40, 600, 2)])
@pytest.mark.parametrize('extra', [1, 3, 6])
def test_backward_with_more_rows_than_images(ops, HW, C, G, extra):
    """the trailing rows of dy belong to the last images once more: as if those images were appended to x, with dgamma / dbeta
    from the first rows only - bit for bit, every image's sums being formed the same way"""
    N = 6
    x, gamma, beta, dy = data(N, HW, C, 11, extra)
    x, gamma, beta, dy = x.cuda(), gamma.cuda(), beta.cuda(), dy.cuda()
    _, stats = ops.group_norm_fwd(x, gamma, beta, G, act='lrelu')
    dx, dg, db = ops.group_norm_bwd(x, dy, gamma, beta, stats, act='lrelu')
    xx, ss = torch.cat([x, x[N - extra:]]), torch.cat([stats, stats[N - extra:]])
    rx, _, _ = ops.group_norm_bwd(xx, dy, gamma, beta, ss, act='lrelu')
    x1, rg, rb = ops.group_norm_bwd(x, dy[:N].contiguous(), gamma, beta, stats, act='lrelu')
    assert torch.equal(dx, rx) and torch.equal(dx[:N], x1)
    assert torch.allclose(dg, rg, rtol=4 * U, atol=1e-6) and torch.allclose(db, rb, rtol=4 * U, atol=1e-6)
    nx, none, none2 = ops.group_norm_bwd(x, dy, gamma, beta, stats, act='lrelu', param_grads=False)
    assert torch.equal(nx, dx) and none is None and none2 is None


def test_sign_next_to_zero_is_the_exact_one(ops):
    """z of a few parts in 2^-24: relu's derivative follows the exact value's sign, as 64 bits decide it"""
    N, HW, C, G = 4, 64, 32, 8
    x, gamma, _, dy = data(N, HW, C, 19)
    _, _, _, xhat = forward64(x.double(), gamma.double(), torch.zeros(C).double(), G, 'linear')
    beta = (-(xhat[0, 5] * gamma.double())).float()              # z of image 0, pixel 5 is beta's rounding error
    _, stats = ops.group_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), G, act='relu')
    dx, dg, db = ops.group_norm_bwd(x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda(), stats, act='relu')
    rx, rg, rb, terms, _, _ = backward64(x.double(), dy.double(), gamma.double(), beta.double(), G, 'relu')
    z = xhat[0, 5] * gamma.double() + beta.double()
    assert (z.abs() < 4 * U).any() and (z.abs() > 1e-12).all()
    assert ((dx.cpu().double() - rx).abs() <= U * rx.abs() + 1e-12 * terms).all()


def test_unaligned_tensors_in_place_and_single_outputs(ops):
    N, HW, C, G = 3, 50, 32, 8
    x, gamma, beta, dy = (t.cuda() for t in data(N, HW, C, 23))
    y, stats = ops.group_norm_fwd(x, gamma, beta, G, act='relu')
    dx, dg, db = ops.group_norm_bwd(x, dy, gamma, beta, stats, act='relu')

    def off_by_one(t):
        b = torch.full((t.numel() + 9,), 7.0, device='cuda')
        v = b[1:1 + t.numel()].view(t.shape)
        v.copy_(t)
        return b, v
    (bx, ux), (bo, uo) = off_by_one(x), off_by_one(x)
    y2, st2 = ops.group_norm_fwd(ux, gamma, beta, G, act='relu', out=uo)
    assert torch.allclose(y2, y, rtol=2 * U, atol=1e-9) and torch.allclose(st2, stats, rtol=1e-12, atol=1e-14)
    assert (bo[0] == 7) and (bo[1 + x.numel():] == 7).all()          # nothing outside the view was written
    z = x.clone()
    y3, _ = ops.group_norm_fwd(z, gamma, beta, G, act='relu', out=z)
    assert torch.equal(y3, y) and y3.data_ptr() == z.data_ptr()
    d = dy.clone()
    dx3, _, _ = ops.group_norm_bwd(x, d, gamma, beta, stats, act='relu', out=d)
    assert torch.equal(dx3, dx)
    for view in ((N, 5, 10, C), (N, HW, C)):                         # pixels in any number of dimensions
        assert torch.equal(ops.group_norm_fwd(x.view(view), gamma, beta, G, act='relu')[0].view_as(y), y)


def test_a_bad_image_stays_its_own(ops):
    """infinities and NaN in one image reach that image's outputs only; a constant image gives beta"""
    N, HW, C, G = 4, 40, 16, 4
    x, gamma, beta, dy = (t.cuda() for t in data(N, HW, C, 29))
    y0, _ = ops.group_norm_fwd(x, gamma, beta, G)
    x2 = x.clone()
    x2[1, 3, 2], x2[3] = float('nan'), 2.5
    x2[2, 0, 9] = float('inf')
    y, stats = ops.group_norm_fwd(x2, gamma, beta, G)
    assert torch.equal(y[0], y0[0]) and torch.isnan(y[1, :, :4]).all() and torch.equal(y[1, :, 4:], y0[1, :, 4:])
    assert torch.isnan(y[2, :, 8:12]).all() and torch.equal(y[2, :, :8], y0[2, :, :8])
    assert torch.allclose(y[3], beta.expand(HW, C)) and torch.isfinite(stats[3]).all()
    dx, _, _ = ops.group_norm_bwd(x2, dy, gamma, beta, stats)
    assert torch.isfinite(dx[0]).all() and torch.isfinite(dx[3]).all()


def test_streams_graphs_and_plans(ops):
    """on another stream, captured in a graph (replayed with eager work between), recorded in a launch plan: the same bits"""
    import ctypes
    from mmdgan_hip import _lib
    for N, HW, C, G in ((8, 64, 64, 8), (4, 50, 30, 5)):
        x, gamma, beta, dy = (t.cuda() for t in data(N, HW, C, 31))
        y, stats = ops.group_norm_fwd(x, gamma, beta, G, act='lrelu')
        dx, dg, db = ops.group_norm_bwd(x, dy, gamma, beta, stats, act='lrelu')
        bufs = [torch.zeros_like(t) for t in (y, stats, dx, dg, db)]
        ws = ops.group_norm_workspace(N, HW, C, G, 'cuda')

        def both():
            ops.group_norm_fwd(x, gamma, beta, G, act='lrelu', out=bufs[0], stats=bufs[1], workspace=ws)
            ops.group_norm_bwd(x, dy, gamma, beta, bufs[1], act='lrelu', out=bufs[2], dgamma=bufs[3], dbeta=bufs[4], workspace=ws)

        def same():
            torch.cuda.synchronize()
            ok = all(torch.equal(a, b) for a, b in zip(bufs, (y, stats, dx, dg, db)))
            for b in bufs:
                b.zero_()
            torch.cuda.synchronize()
            return ok
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            both()
        assert same()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            both()
        same()
        for _ in range(3):
            graph.replay()
            assert same()
            ops.group_norm_fwd(x, gamma, beta, G, act='relu')
        lib = _lib.load()
        handle = ops.Handle(workspace_bytes=0)
        with handle:
            ops.check(lib.mmdgan_plan_begin(), 'plan_begin')
            both()
            pid = ctypes.c_int(-1)
            ops.check(lib.mmdgan_plan_end(ctypes.byref(pid)), 'plan_end')
            assert same()
            for _ in range(2):
                ops.check(lib.mmdgan_plan_replay(pid.value, -1), 'plan_replay')
                assert same()
            names = {k[0] for k in ops.plan_kernels(pid.value)}
            assert all(n.startswith('gn_') for n in names), names


def test_offsets_past_32_bits(ops):
    """a batch of more than 2^31 values: the last image like the first"""
    N, HW, C, G = 2200, 16384, 64, 8
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip('needs 30 GB of device memory')
    one = torch.randn(1, HW, C, device='cuda')
    gamma, beta = torch.rand(C, device='cuda') + 0.5, torch.randn(C, device='cuda')
    x = torch.zeros(N, HW, C, device='cuda')
    x[0], x[N - 1] = one[0], one[0]
    y, stats = ops.group_norm_fwd(x, gamma, beta, G, act='relu', out=x)
    assert torch.equal(y[0], y[N - 1]) and torch.equal(stats[0], stats[N - 1])
    r, _ = ops.group_norm_fwd(one, gamma, beta, G, act='relu')
    assert torch.allclose(y[N - 1], r[0], rtol=4 * U, atol=1e-7) and float(y[N // 2].max()) == float(beta.clamp(min=0).max())


def test_refusals_on_the_device(ops):
    x, gamma, beta, dy = (t.cuda() for t in data(2, 9, 12, 37))
    y, stats = ops.group_norm_fwd(x, gamma, beta, 3)
    with pytest.raises(ValueError, match='do not divide'):
        ops.group_norm_fwd(x, gamma, beta, 5, stats=torch.empty(2, 5, 2, device='cuda', dtype=torch.float64),
                           workspace=torch.empty(1 << 16, device='cuda', dtype=torch.uint8))
    with pytest.raises(NotImplementedError):
        ops.group_norm_fwd(x, gamma, beta, 3, act='selu')
    with pytest.raises(AssertionError):
        ops.group_norm_fwd(x.half(), gamma, beta, 3)
    with pytest.raises(AssertionError):
        ops.group_norm_fwd(x.transpose(1, 2), gamma, beta, 3)
    with pytest.raises(AssertionError):
        ops.group_norm_fwd(x, gamma, beta, 3, stats=torch.empty(2, 3, 2, device='cuda'))
    with pytest.raises(AssertionError, match='workspace'):
        ops.group_norm_fwd(x, gamma, beta, 3, workspace=torch.empty(8, device='cuda', dtype=torch.uint8))
    with pytest.raises(ValueError, match='x_batch'):
        ops.group_norm_bwd(x, torch.cat([dy, dy, dy]), gamma, beta, stats)
    with pytest.raises(ValueError, match='eps'):
        ops.group_norm_fwd(x, gamma, beta, 3, eps=0.0)


def test_a_workspace_is_real_memory(ops):
    """an expanded tensor counts more bytes than it has"""
    x, v = torch.randn(2, 9, 12, device='cuda'), torch.ones(12, device='cuda')
    fake = torch.zeros(1, device='cuda', dtype=torch.uint8).expand(1 << 20)
    y, st = ops.group_norm_fwd(x, v, v, 3)
    with pytest.raises(AssertionError, match='workspace'):
        ops.group_norm_fwd(x, v, v, 3, workspace=fake)
    with pytest.raises(AssertionError, match='workspace'):
        ops.group_norm_bwd(x, x, v, v, st, workspace=fake)


@pytest.mark.parametrize('N,HW,C,G', [(4, 40, 16, 4), (4, 40, 16, 16), (3, 50, 60, 12), (3, 35, 15, 5), (2, 3000, 12, 4)])
def test_a_bad_image_shows_under_every_activation(ops, N, HW, C, G):
    """a group that holds an infinity or NaN is NaN in y whatever the activation (relu of NaN is NaN), as in dx; the other groups and images
    keep their bits"""
    x, gamma, beta, dy = (t.cuda() for t in data(N, HW, C, 41))
    D = C // G
    for act in ('linear', 'relu', 'lrelu', 'tanh'):
        y0, st0 = ops.group_norm_fwd(x, gamma, beta, G, act=act)
        dx0, _, _ = ops.group_norm_bwd(x, dy, gamma, beta, st0, act=act)
        for bad in (float('nan'), float('inf'), float('-inf')):
            x2 = x.clone()
            x2[1, HW // 2, D] = bad                              # image 1, group 1
            y, st = ops.group_norm_fwd(x2, gamma, beta, G, act=act)
            dx, _, _ = ops.group_norm_bwd(x2, dy, gamma, beta, st, act=act)
            spoiled = torch.zeros_like(y, dtype=torch.bool)
            spoiled[1, :, D:2 * D] = True
            assert torch.equal(torch.isnan(y), spoiled) and torch.equal(torch.isnan(dx), spoiled), (act, bad)
            assert torch.equal(y[~spoiled], y0[~spoiled]) and torch.equal(dx[~spoiled], dx0[~spoiled])


@pytest.mark.parametrize('N,HW,C,G', [(3, 65, 48, 12), (2, 1023, 32, 8), (3, 64, 32, 32), (3, 50, 60, 12), (2, 33, 15, 5), (2, 9000, 4, 4), (33, 1457, 96, 32)])
def test_tanh_backward_within_its_own_error(ops, N, HW, C, G):
    """the slope is 4 e / (1 + e)^2 with e = exp(-2 |z|) in 32 bits.  e: (2 + 6 |z|) u (the exponential's last place is 2 u; z, the constant and
    their product u each, of 2 |z|), of which tanh |z| counts, times the slope 1 / cosh^2 z: at most 2.6 u.  1 + e: u, its reciprocal 2 u, both
    squared, and two products: 8 u of the slope.  Together at most 9 u of 1; dz itself stays in 64 bits.  So dx is within u of itself and 9 u
    of each term |rstd gamma dy| (2 + |xhat|), and the parameters' sums within 9 u of theirs."""
    x, gamma, beta, dy = data(N, HW, C, 51 + C)
    _, stats = ops.group_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), G, act='tanh')
    dx, dgamma, dbeta = ops.group_norm_bwd(x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda(), stats, act='tanh')
    rx, rg, rb, terms, dz, xhat = backward64(x.double(), dy.double(), gamma.double(), beta.double(), G, 'tanh')
    z = torch.linspace(0, 20, 1 << 16, dtype=torch.float64)
    assert float(((2 + 6 * z) * torch.tanh(z) / torch.cosh(z) ** 2 + 8 / torch.cosh(z) ** 2).max()) <= 9
    slack = 9 * U
    assert ((dx.cpu().double() - rx).abs() <= U * rx.abs() + (slack + 1e-11) * terms).all()
    a = dy.double().abs()
    assert ((dgamma.cpu().double() - rg).abs() <= U * rg.abs() + (slack + 1e-11) * (a * xhat.abs()).sum(dim=(0, 1))).all()
    assert ((dbeta.cpu().double() - rb).abs() <= U * rb.abs() + (slack + 1e-11) * a.sum(dim=(0, 1))).all()
