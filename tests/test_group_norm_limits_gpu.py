"""Group norm at the largest image that its entries take: HW * C just below 2^31, where rows counted from the image's start pass an int.
Tolerances as in test_group_norm_gpu.py: a result is the exact value rounded once (u = 2^-24), dx up to 1e-12 of its terms for the sums
of 2^31 values in 64 bits (2^31 roundings of 2^-53 at random signs: 2^-37 of a term, 7e-12 at the very worst of all of one sign)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEP = 1 << 26


@pytest.fixture(scope='module')
def ops():
    from mmdgan_hip import ops as o
    o.require_device()
    return o


def pieces(n):
    return [slice(i, min(i + STEP, n)) for i in range(0, n, STEP)]


@pytest.mark.parametrize('HW,C,G', [(0x7fffffff, 1, 1), (0x7fffffff // 3, 3, 3), (0x7fffffff // 4, 4, 1)])
def test_the_largest_image(ops, HW, C, G):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of device memory')
    g = torch.Generator(device='cuda').manual_seed(HW % 1000)
    x = torch.empty(1, HW, C, device='cuda').normal_(generator=g)
    x[0, -(HW // 64):] += 3.0                               # the last chunk is not like the others
    gamma, beta = torch.rand(C, device='cuda', generator=g) + 0.5, torch.randn(C, device='cuda', generator=g)
    y, stats = ops.group_norm_fwd(x, gamma, beta, G, act='lrelu')
    D, rows = C // G, x[0]
    total = lambda f: sum(f(rows[s].double()).view(-1, G, D).sum(dim=(0, 2)) for s in pieces(HW))
    mean = total(lambda v: v) / (HW * D)
    per = lambda t: t.repeat_interleave(D)
    rstd = 1 / torch.sqrt(total(lambda v: (v - per(mean)) ** 2) / (HW * D) + float(torch.tensor(1e-5)))
    assert torch.allclose(stats[0, :, 0], mean, rtol=1e-11, atol=1e-11) and torch.allclose(stats[0, :, 1], rstd, rtol=1e-11)
    hat = lambda s: (rows[s].double() - per(mean)) * per(rstd)
    for s in pieces(HW):
        z = hat(s) * gamma.double() + beta.double()
        ref = torch.where(z > 0, z, 0.1 * z)
        assert ((y[0, s].double() - ref).abs() <= 3 * U * ref.abs() + 1e-10).all(), s
    del y
    dy = torch.empty_like(x).normal_(generator=g)
    dx, dgamma, dbeta = ops.group_norm_bwd(x, dy, gamma, beta, stats, act='lrelu')
    dz = lambda s: dy[0, s].double() * torch.where(hat(s) * gamma.double() + beta.double() > 0, 1.0, float(torch.tensor(0.1)))
    sums = [(dz(s).sum(dim=0), (dz(s) * hat(s)).sum(dim=0), dz(s).abs().sum(dim=0)) for s in pieces(HW)]
    b, gm, size = (sum(t) for t in zip(*sums))
    assert ((dbeta.double() - b).abs() <= U * b.abs() + 1e-11 * size).all()
    assert ((dgamma.double() - gm).abs() <= U * gm.abs() + 1e-10 * size).all()
    group = lambda t: per((t * gamma.double()).view(G, D).sum(dim=1) / (HW * D))
    m1, m2 = group(b), group(gm)
    for s in pieces(HW):
        t = dz(s) * gamma.double()
        ref = per(rstd) * (t - m1 - hat(s) * m2)
        assert ((dx[0, s].double() - ref).abs() <= U * ref.abs() + 1e-10 * (1 + t.abs())).all(), s


def test_many_one_channel_groups(ops):
    """2^22 - 1 groups of one value: each is its own mean, and y is beta but for A x + B = rstd gamma x + (beta - rstd gamma x): B and the sum
    are rounded to 64 bits, 2^-53 of |beta| + |rstd gamma x| each (|x| rstd being at most 256 where B is not taken around x itself), before
    one rounding to 32"""
    C = (1 << 22) - 1
    g = torch.Generator(device='cuda').manual_seed(3)
    x, gamma, beta = (torch.randn(C, device='cuda', generator=g) for _ in range(3))
    y, stats = ops.group_norm_fwd(x.view(1, 1, C), gamma, beta, C)
    assert torch.equal(stats[0, :, 0], x.double())
    b = beta.double().abs()
    assert ((y.view(-1).double() - beta.double()).abs() <= U * b + 2 * 2.0 ** -53 * (b + 256 * gamma.double().abs())).all()
