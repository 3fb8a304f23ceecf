"""Group norm of values whose mean is far from zero, measured in their standard deviations: biased images, constant groups.

Bars (e = 2^-53, u = 2^-24), none of which grows with mean^2.  With k the group's first value and q = E[(x - k)^2] rstd^2 <= M: the sums around
k lose 64 roundings of e q of the variance (a few dozen additions in sequence; the rest are tree sums), the sums around zero, which are
kept while |mean| rstd <= 256, 64 e 2^16.  So rstd is good to d = 32 e (q + 2^16), relatively, and the mean to e |mean| for its own
rounding and 64 e sqrt(q) / rstd, or 64 e 2^8 / rstd, for the sum's.  With c the mean rounded to 32 bits, x - c is exact for x between c / 2 and
2 c, else off by u |x - c|, half a step.  z = (x - mean) rstd gamma + beta is then off by (m rstd + d |xhat| + u |xhat| [far]) |gamma|, m the
error of the mean, and rounded once.  In dx and the parameters' sums the same errors enter linearly; means are at most the largest term."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -24, 2.0 ** -53
EPS = float(np.float32(1e-5))

# resident forms (four channels of one group, of several; no power of two), one and several images a workgroup; two passes with vector and
# scalar loads, groups wider than a slab
GEOMETRIES = [(4, 64, 64, 8), (2, 1024, 64, 4), (2, 4096, 64, 16), (3, 100, 32, 16), (2, 1000, 64, 64), (3, 77, 60, 12), (5, 100, 48, 4), (2, 600, 160, 32),
              (1100, 3, 12, 4), (2, 1457, 96, 32), (2, 130, 254, 127), (3, 700, 3, 1), (2, 20, 768, 1), (1, 3, 1031, 1), (2, 40, 1200, 2), (2500, 1, 128, 4)]
LRELU = float(np.float32(0.1))


@pytest.fixture(scope='module')
def ops():
    from mmdgan_hip import ops as o
    o.require_device()
    return o


def statistics(x, G):
    """mean, rstd, q of every group, from differences to the group's first value (exact in 64 bits where they matter)"""
    N, HW, C = x.shape
    v = x.double().view(N, HW, G, C // G)
    k = v[:, 0, :, 0].view(N, 1, G, 1)
    d = v - k
    off = d.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((d - off).square().mean(dim=(1, 3), keepdim=True) + EPS)
    return k + off, rstd, d.square().mean(dim=(1, 3), keepdim=True) * rstd ** 2, (d - off) * rstd


def check(ops, x, G, act, seed):
    N, HW, C = x.shape
    g = torch.Generator().manual_seed(seed)
    gamma, beta = (1 + 0.3 * torch.randn(C, generator=g)).float(), (0.3 * torch.randn(C, generator=g)).float()
    dy = torch.randn(N, HW, C, generator=g).float()
    mean, rstd, q, xhat = statistics(x, G)
    y, stats = ops.group_norm_fwd(x.cuda(), gamma.cuda(), beta.cuda(), G, act=act)
    st = stats.cpu().view(N, 1, G, 1, 2)
    d = 32 * E * (q + 2.0 ** 16)
    m = E * mean.abs() + 64 * E * torch.maximum(q.sqrt(), torch.tensor(256.0)) / rstd
    assert torch.isfinite(st).all()
    assert ((st[..., 0] - mean).abs() <= m).all(), float(((st[..., 0] - mean).abs() / m).max())
    assert ((st[..., 1] - rstd).abs() <= d * rstd).all(), float(((st[..., 1] / rstd - 1).abs() / d).max())
    outside = (x.double().view(xhat.shape) / mean - 1.25).abs() > 0.75
    far = U * (outside & (mean.abs() * rstd > 200)).double()
    err = (m * rstd + (d + far) * xhat.abs()).reshape(N, HW, C)                        # of xhat
    hat = xhat.reshape(N, HW, C)
    gm, bt = gamma.double(), beta.double()
    z = hat * gm + bt
    below = {'linear': 1.0, 'relu': 0.0, 'lrelu': LRELU}[act]
    ref = torch.where(z > 0, z, below * z)
    assert ((y.cpu().double() - ref).abs() <= (3 if act == 'lrelu' else 1) * U * ref.abs() + err * gm.abs() + 1e-13).all()
    # backward, from the kernel's statistics; elements whose sign the forward error could turn are left out of nothing: there are none
    assert (z.abs() > err * gm.abs()).all() or act == 'linear'
    dx, dgamma, dbeta = ops.group_norm_bwd(x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda(), stats, act=act)
    dz = dy.double() * torch.where(z > 0, 1.0, below)
    t, p = (dz * gm).view(xhat.shape), xhat
    rx = rstd * (t - t.mean(dim=(1, 3), keepdim=True) - p * (t * p).mean(dim=(1, 3), keepdim=True))
    big = (dy.double() * gm).abs().view(xhat.shape).amax(dim=(1, 3), keepdim=True)
    e = err.view(xhat.shape)
    emax, pmax = e.amax(dim=(1, 3), keepdim=True), p.abs().amax(dim=(1, 3), keepdim=True)
    tol = rstd * big * (1e-13 + d * (2 + p.abs() * p.abs().mean(dim=(1, 3), keepdim=True)) + e * p.abs().mean(dim=(1, 3), keepdim=True) + p.abs() * emax)
    assert ((dx.cpu().double().view(xhat.shape) - rx).abs() <= U * rx.abs() + tol).all()
    a = dz.abs()
    rg, rb = (dz * hat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    assert ((dgamma.cpu().double() - rg).abs() <= U * rg.abs() + (a * (err + 1e-13 * (1 + hat.abs()))).sum(dim=(0, 1)) + 1e-30).all()
    assert ((dbeta.cpu().double() - rb).abs() <= U * rb.abs() + 1e-13 * a.sum(dim=(0, 1))).all()


@pytest.mark.parametrize('N,HW,C,G', GEOMETRIES)
def test_means_far_from_zero(ops, N, HW, C, G):
    """from one standard deviation to beyond what 32 bits resolve of a value"""
    g = torch.Generator().manual_seed(HW + C)
    r = torch.randn(N, HW, C, generator=g, dtype=torch.float64)
    for i, (mean, std) in enumerate(((1.0, 1.0), (30.0, 1.0), (-500.0, 1.0), (1e4, 1.0), (1e5, 1.0), (-1000.0, 1e-2), (1e4, 1e-2), (1e6, 1.0), (3e5, 0.05))):
        print(N, HW, C, G, mean, std, flush=True)
        check(ops, (mean + std * r).float(), G, ('linear', 'lrelu', 'relu')[i % 3], i)


@pytest.mark.parametrize('N,HW,C,G', GEOMETRIES)
def test_images_of_different_means(ops, N, HW, C, G):
    """near and far groups, channels and images in one call: each by its own rule"""
    g = torch.Generator().manual_seed(HW)
    r = torch.randn(N, HW, C, generator=g, dtype=torch.float64)
    shift = torch.tensor([0.0, 300.0, 1e5, -1e4])[torch.randint(0, 4, (N, 1, G, 1), generator=g)].double()
    check(ops, (r.view(N, HW, G, -1) + shift).view(N, HW, C).float(), G, 'lrelu', 3)
    x = r + 5
    x[:, 0, :] = 2000.0                                     # the first value itself is the outlier
    check(ops, x.float(), G, 'linear', 4)


@pytest.mark.parametrize('N,HW,C,G', GEOMETRIES)
def test_constant_groups(ops, N, HW, C, G):
    """their variance is 0: y is act(beta) exactly (x - mean is), rstd is 1 / sqrt(eps) - also in place, and beside groups that vary"""
    g = torch.Generator().manual_seed(7)
    gamma, beta = torch.rand(C, generator=g).cuda() + 0.5, torch.randn(C, generator=g).cuda()
    dy = torch.randn(N, HW, C, generator=g).cuda()
    for value in (0.0, 0.1, -7.3, 3e5, 1e8, -1e30, 3e38):
        x = torch.full((N, HW, C), value).float().cuda()
        y, stats = ops.group_norm_fwd(x, gamma, beta, G, act='relu')
        assert torch.equal(stats[..., 0], x[:, 0, ::C // G].double()), value
        # (|mean| rstd <= 256 around zero: the difference of 64 e mean^2 against eps)
        assert torch.allclose(stats[..., 1], torch.tensor(EPS ** -0.5, dtype=torch.float64), rtol=32 * E * 2 ** 16, atol=0), value
        assert torch.allclose(y, beta.clamp(min=0).expand_as(y), rtol=2 * U, atol=1e-12), value
        z = x.clone()
        assert torch.equal(ops.group_norm_fwd(z, gamma, beta, G, act='relu', out=z)[0], y)
        # xhat is 0: dx = rstd (gamma dy - mean(gamma dy)), dgamma = 0
        dx, dgamma, dbeta = ops.group_norm_bwd(x, dy, gamma, beta, stats)
        t = (dy.double() * gamma.double()).view(N, HW, G, -1)
        ref = (EPS ** -0.5 * (t - t.mean(dim=(1, 3), keepdim=True))).view(N, HW, C)
        scale = float(ref.abs().max()) + EPS ** -0.5 * float(t.abs().max())
        assert ((dx.double() - ref).abs() <= 2 * U * ref.abs() + 1e-10 * scale).all(), value
        assert (dgamma.double().abs() <= 1e-10 * dy.double().abs().sum(dim=(0, 1))).all(), value


def test_infinities_and_nan_in_the_first_value(ops):
    """the value that a group's sums may be taken around: its image's group is spoiled, as by any other, and nothing else"""
    for N, HW, C, G in ((3, 64, 32, 8), (3, 64, 32, 32), (3, 50, 60, 12), (3, 30, 15, 5), (3, 3000, 12, 4), (2, 9, 600, 2)):
        g = torch.Generator().manual_seed(3)
        x = (torch.randn(N, HW, C, generator=g) + 2000).cuda()
        gamma, beta = torch.ones(C, device='cuda'), torch.zeros(C, device='cuda')
        y0, s0 = ops.group_norm_fwd(x, gamma, beta, G)
        for bad in (float('inf'), float('-inf'), float('nan')):
            x2 = x.clone()
            x2[1, 0, 0] = bad
            y, s = ops.group_norm_fwd(x2, gamma, beta, G)
            D = C // G
            assert torch.isnan(y[1, :, :D]).all() and torch.isnan(s[1, 0, 1])
            keep = torch.ones(N, C, dtype=torch.bool)
            keep[1, :D] = False
            assert torch.equal(y.permute(0, 2, 1)[keep.cuda()], y0.permute(0, 2, 1)[keep.cuda()])
            ks = torch.ones(N, G, dtype=torch.bool)
            ks[1, 0] = False
            assert torch.equal(s[ks.cuda()], s0[ks.cuda()])


def test_in_place_far_from_zero(ops):
    """y on x, dx on dy and on x: the second reading of x comes before anything is written"""
    for N, HW, C, G in GEOMETRIES:
        g = torch.Generator().manual_seed(C)
        x = (torch.randn(N, HW, C, generator=g) + 1e5).cuda()
        gamma, beta, dy = torch.rand(C, generator=g).cuda(), torch.randn(C, generator=g).cuda(), torch.randn(N, HW, C, generator=g).cuda()
        y, st = ops.group_norm_fwd(x, gamma, beta, G, act='relu')
        dx, dg, db = ops.group_norm_bwd(x, dy, gamma, beta, st, act='relu')
        for _ in range(3):
            z = x.clone()
            y2, st2 = ops.group_norm_fwd(z, gamma, beta, G, act='relu', out=z)
            assert torch.equal(y2, y) and torch.equal(st2, st), (N, HW, C, G)
        d = dy.clone()
        assert torch.equal(ops.group_norm_bwd(x, d, gamma, beta, st, act='relu', out=d)[0], dx)
        z = x.clone()
        assert torch.equal(ops.group_norm_bwd(z, dy, gamma, beta, st, act='relu', out=z)[0], dx)


@pytest.mark.parametrize('extra', [1, 3])
def test_more_rows_than_images_far_from_zero(ops, extra):
    """dy's trailing rows read the last images' values and statistics once more, in every form of the backward pass"""
    N = 4
    for HW, C, G in ((64, 32, 8), (64, 32, 32), (64, 32, 16), (50, 60, 12), (37, 15, 5), (1500, 96, 32), (20, 768, 1)):
        for shift in (0.0, 1e5):
            g = torch.Generator().manual_seed(C)
            x = (torch.randn(N, HW, C, generator=g) + shift).cuda()
            gamma, beta, dy = torch.rand(C, generator=g).cuda(), torch.randn(C, generator=g).cuda(), torch.randn(N + extra, HW, C, generator=g).cuda()
            _, st = ops.group_norm_fwd(x, gamma, beta, G)
            dx, dg, db = ops.group_norm_bwd(x, dy, gamma, beta, st, act='lrelu')
            rx, _, _ = ops.group_norm_bwd(torch.cat([x, x[N - extra:]]), dy, gamma, beta, torch.cat([st, st[N - extra:]]), act='lrelu')
            x1, rg, rb = ops.group_norm_bwd(x, dy[:N].contiguous(), gamma, beta, st, act='lrelu')
            assert torch.equal(dx, rx) and torch.equal(dx[:N], x1), (HW, C, G, shift)
            assert torch.allclose(dg, rg, rtol=4 * U, atol=1e-5) and torch.allclose(db, rb, rtol=4 * U, atol=1e-5)
