"""Orthogonalisation at every allowed number of steps on matrices that have next to nothing along some directions: rank one, low
rank, six decades of singular values.  Rounding puts a little along such a direction, and the polynomial multiplies it by
3.44 a step; it has to settle where p takes every singular value and must not grow past it.

p(s) = a s + b s^3 + c s^5 maps [0, 1.2637] into itself: p' = 0 at s^2 = 0.3075 and 1.1028, where p is 1.20237 (its maximum up to
s = 1.25) and 0.682, and p(s) = s at 1.2637.  So with TOP = 1.20237 and d the error of one Gram-to-Gram stretch, singular values of at
most TOP + d go to at most TOP, plus d once more, while d < 0.04.  d in the spectral norm, which the Frobenius norm bounds: with sides above 64 a
stretch is three steps of products held to 2 * 2^-23 of norms of at most 1.25 sqrt(m), each error stretched by at most a by the steps
behind it: (1 + a + a^2) * 2 * 2^-23 * 1.25 sqrt(m) = 41 * 2^-23 sqrt(m).  With a side of 64 or less eight steps in 64 bits and one rounding to 32,
which is less.
"""
import math

import pytest
import torch

from test_muon_gpu import A, B, C, make, orth64, tolerance

pytestmark = pytest.mark.gpu

TOP = 1.202369          # max of p on [0, 1.25] (1.2023686), rounded up
SHAPES = [(32, 288), (16, 1024), (576, 64), (2304, 64), (1, 40), (260, 150), (65, 900)]
KINDS = ('rank1', 'lowrank', 'decay', 'normal', 'gradient')


def p(s):
    return A * s + B * s ** 3 + C * s ** 5


def dp(s):
    return A + 3 * B * s ** 2 + 5 * C * s ** 4


def stretch_error(m):
    return 41 * 2.0 ** -23 * math.sqrt(m)


@pytest.fixture(scope='module')
def ops():
    from mmdgan_hip import ops as o
    o.require_device()
    return o


def test_the_bound_itself():
    s = torch.linspace(0, 1.25, 1 << 20, dtype=torch.float64)
    assert float(p(s).max()) <= TOP and abs(float(p(s).max()) - TOP) < 1e-6


@pytest.mark.parametrize('steps', list(range(1, 17)))
def test_singular_values_stay_bounded_at_any_number_of_steps(ops, steps):
    for rows, cols in SHAPES:
        us = [make(kind, rows, cols, 31 * steps + i) for i, kind in enumerate(KINDS)]
        outs = ops.orthogonalize([u.cuda() for u in us], steps=steps)
        for kind, u, o in zip(KINDS, us, outs):
            o = o.cpu().double()
            assert torch.isfinite(o).all(), (rows, cols, kind)
            top = float(torch.linalg.matrix_norm(o, 2))
            assert top <= TOP + stretch_error(min(rows, cols)) + 2.0 ** -24 * float(o.norm()), (rows, cols, kind, top)


@pytest.mark.parametrize('steps', [5, 8, 9, 12, 16])
def test_the_leading_direction_follows_the_polynomial(ops, steps):
    """u^T O v of a rank-one matrix: its one singular value, 1 after the normalisation, along p's orbit.  An error e in s becomes
    max |p'| e over [s - e, s + e]; a step adds what a stretch does, at most.  (Errors off the diagonal change it in second order.)"""
    for rows, cols in SHAPES:
        u = make('rank1', rows, cols, steps)
        o = ops.orthogonalize(u.cuda(), steps=steps).cpu().double()
        left, s, right = torch.linalg.svd(u.double(), full_matrices=False)
        x, e, d = float(s[0] / s.norm()), 2.0 ** -22, stretch_error(min(rows, cols))
        for _ in range(steps):
            grid = torch.linspace(x - e, x + e, 101, dtype=torch.float64)
            e = float(dp(grid).abs().max()) * e + d
            x = p(x)
        got = float(left[:, 0] @ o @ right[0])
        assert e < 0.2 and abs(got - x) <= e, (rows, cols, got, x, e)


@pytest.mark.parametrize('nesterov', [True, False])
def test_an_update_of_many_steps_is_its_orthogonalised_momentum(ops, nesterov):
    """the update's O at 9 and 16 steps is orthogonalize's of the momentum, whose scratch also holds the iterate; momentum kept"""
    for steps in (8, 9, 16):
        for rows, cols in ((32, 288), (1024, 16), (64, 64), (130, 70)):
            g = make('lowrank', rows, cols, steps).cuda()
            p0, m0 = torch.zeros(rows, cols, device='cuda'), torch.zeros(rows, cols, device='cuda')
            ps, ms = p0.clone(), m0.clone()
            ops.MuonGroup([ps], [g], [ms]).step(1.0, momentum=0.0, nesterov=nesterov, steps=steps)
            o = ops.orthogonalize(g, steps=steps)            # (momentum 0: U = g)
            c = float(torch.tensor(0.2 * math.sqrt(max(rows, cols)), dtype=torch.float32))
            assert torch.equal(ms, g)
            # (both sides round the same O, times c, to 32 bits: two roundings apart)
            assert ((ps.double() + c * o.double()).abs() <= 2 * 2.0 ** -24 * c * o.double().abs() + 1e-30).all(), (rows, cols, steps)


def test_many_steps_in_place_in_a_graph_and_with_foreign_scratch(ops):
    us = [make('rank1', r, c, i).cuda() for i, (r, c) in enumerate([(32, 288), (1024, 16), (64, 64), (3, 5), (130, 70)])]
    want = ops.orthogonalize(us, steps=16)
    need = ops.orthogonalize_workspace(us, steps=16).numel()
    ws = torch.full((need + 4096,), 0x55, device='cuda', dtype=torch.uint8)
    outs = [u.clone() for u in us]
    ops.orthogonalize(outs, steps=16, out=outs, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and (ws[need:] == 0x55).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.orthogonalize(us, steps=16, out=outs, workspace=ws)
    for _ in range(3):
        for o in outs:
            o.zero_()
        ops.orthogonalize(us[::-1], steps=9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 6, 7])
def test_few_steps_on_matrices_of_every_kind(ops, steps):
    """against the definition at test_muon_gpu.py's bar, a score of matrices of each kind: the bar is tight at few steps, where nothing has been
    stretched yet, and rank-one matrices with a long side come nearest to it"""
    for rows, cols in ((66, 271), (4000, 70), (129, 300), (40, 300)):
        for kind in KINDS:
            us = [make(kind, rows, cols, seed) for seed in [48244] + list(range(1000 * steps, 1000 * steps + 20))]
            outs = ops.orthogonalize([u.cuda() for u in us], steps=steps)
            for u, o in zip(us, outs):
                ref = orth64(u, steps)
                err, bar = float((o.cpu().double() - ref).norm()), tolerance(u, ref, steps)
                assert err <= bar, (rows, cols, kind, err, bar)
