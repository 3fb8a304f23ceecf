"""Orthogonalisation of matrices and the parameter update that applies it (mmdgan_orthogonalize, mmdgan_muon_update) against the
definition in 64 bits.

Tolerance, in the Frobenius norm.  X0, the Gram matrices, the polynomials, their products and the products with X are held to 2^-23
or better of matrices whose norms are at most those of X: two such roundings for X0 and two per step on the longest way, each
relative to |X_k|_F <= min(a^k, 1.25 sqrt(m)).  A step stretches what errors there are by |p'(s)| at most: p(s) = a s + b s^3 + c s^5
has p' <= a = 3.4445, and once a direction has reached the band that p maps into itself (s from 0.5 to 1.25), |p'| <= 1.61 (p' = a +
3 b s^2 + 5 c s^4 is least at s^2 = 0.705: 3.4445 - 10.10 + 5.05 = -1.61; at 0.5: 3.4445 - 3.58 + 0.63 = 0.50; at 1.25: -22.38 + 24.80 +
3.44 = 5.86 is not reached: the largest image of the band is 1.21, with 3.4445 - 20.97 + 21.77 = 4.24 for that one value, whose own
image is near 0.94 - so a pair of steps stretches by 4.24 * 1.61 < 2.62^2).  So: factor a below 0.5, 2.62 in the band.  The result's own
rounding adds 2^-24 |O|.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope='module')
def ops():
    from mmdgan_hip import ops as o
    o.require_device()
    return o


def orth64(u, steps=5):
    """the definition, doubles, on the side of the columns or rows that is shorter"""
    u = u.double()
    norm = u.norm()
    x = u / norm if norm > 0 else u
    t = x if x.shape[0] <= x.shape[1] else x.t()
    for _ in range(steps):
        k = t @ t.t()
        t = A * t + B * (k @ t) + C * (k @ (k @ t))
    return t if x.shape[0] <= x.shape[1] else t.t()


def tolerance(u, ref, steps=5):
    s = torch.linalg.svdvals(u.double())
    least = float(s[-1] / s.square().sum().sqrt())
    err, norm, top = 2 * 2.0 ** -23, 1.0, 1.25 * math.sqrt(len(s))
    for _ in range(steps):
        err *= A if least < 0.5 else 2.62
        least = A * least + B * least ** 3 + C * least ** 5
        norm = min(norm * A, top)
        err += 2 * 2.0 ** -23 * norm
    return err + 2.0 ** -24 * float(ref.norm())


def make(kind, rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    m, n = min(rows, cols), max(rows, cols)
    r = lambda *s: torch.randn(*s, generator=g)
    if kind == 'normal':
        u = r(m, n)
    elif kind == 'decay':                                  # singular values over six decades
        q, _ = torch.linalg.qr(r(m, m).double())
        w, _ = torch.linalg.qr(r(n, m).double())
        u = ((q * 10 ** torch.linspace(0, -6, m).double()) @ w.t()).float()
    elif kind == 'lowrank':
        k = max(1, m // 4)
        u = r(m, k) @ r(k, n)
    elif kind == 'rank1':
        u = r(m, 1) @ r(1, n)
    else:                                                  # a weight gradient's: decaying, over a floor
        k = max(1, m // 2)
        u = 1e-4 * ((r(m, k) / torch.arange(1, k + 1)) @ r(k, n) + 1e-2 * r(m, n))
    return (u if rows <= cols else u.t().contiguous()).contiguous()


SHAPES = [(1, 1), (1, 17), (33, 1), (2, 3), (27, 64), (64, 27), (8, 27), (16, 1024), (1024, 16), (64, 64), (65, 64), (64, 65), (63, 2000), (31, 4000),
          (128, 128), (129, 1001), (1001, 129), (130, 127), (127, 130), (300, 257), (96, 513), (1024, 200), (257, 2305), (513, 520)]


@pytest.mark.parametrize('rows,cols', SHAPES)
def test_orthogonalize_matches_the_definition(ops, rows, cols):
    for i, kind in enumerate(('normal', 'decay', 'lowrank', 'rank1', 'gradient')):
        u = make(kind, rows, cols, 100 * i + rows)
        print(rows, cols, kind, flush=True)
        ref = orth64(u)
        o = ops.orthogonalize(u.cuda()).cpu().double()
        assert o.shape == u.shape
        err = float((o - ref).norm())
        assert err <= tolerance(u, ref), (kind, err, tolerance(u, ref))


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 6, 7, 10, 16])
def test_any_number_of_steps(ops, steps):
    for rows, cols in ((40, 200), (260, 150)):
        u = make('normal', rows, cols, steps)
        ref = orth64(u, steps)
        o = ops.orthogonalize(u.cuda(), steps=steps).cpu().double()
        assert float((o - ref).norm()) <= tolerance(u, ref, steps)


def test_singular_values_end_near_one(ops):
    u = make('normal', 200, 900, 1).cuda()
    s = torch.linalg.svdvals(ops.orthogonalize(u).double())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.25


def test_scale_zero_and_bad_values(ops):
    for rows, cols in ((40, 90), (200, 140)):
        u = make('normal', rows, cols, 3).cuda()
        o = ops.orthogonalize(u)
        for e in (-100, -20, 60, 100):                     # (a power of two: the normalised matrix is the same, bit for bit)
            assert torch.equal(ops.orthogonalize(torch.ldexp(u, torch.tensor(e, device='cuda'))), o)
        z = torch.zeros_like(u)
        n, f = u.clone(), u.clone()
        n[3, 5], f[1, 1] = float('nan'), float('inf')
        got = ops.orthogonalize([u, z, n, u, f])
        assert torch.equal(got[0], o) and torch.equal(got[3], o)
        assert torch.equal(got[1], z)
        assert torch.isnan(got[2]).any() and torch.isnan(got[4]).any()
        tiny = make('normal', rows, cols, 3) * 1e-42       # subnormal floats: still normalised by their own norm
        ref = orth64(tiny)
        assert float((ops.orthogonalize(tiny.cuda()).cpu().double() - ref).norm()) <= tolerance(tiny, ref)


def test_lists_and_views(ops):
    """many matrices in one call (more than one launch's table holds) give what each gives alone; a conv kernel is its matrix view"""
    shapes = [(27, 16), (3, 3), (144, 32), (40, 300), (300, 150), (1, 9)] * 6
    us = [make('normal', r, c, i).cuda() for i, (r, c) in enumerate(shapes)]
    together = ops.orthogonalize(us)
    for u, o in zip(us, together):
        assert torch.equal(ops.orthogonalize(u), o)
    k = torch.randn(3, 3, 20, 70, device='cuda')
    assert torch.equal(ops.orthogonalize(k).view(180, 70), ops.orthogonalize(k.view(180, 70)))
    v = [u.clone() for u in us]
    ops.orthogonalize(v, out=v)                            # in place
    assert all(torch.equal(a, b) for a, b in zip(v, together))
    assert ops.orthogonalize([]) == []


def test_nothing_outside_the_outputs_is_written(ops):
    for rows, cols in ((27, 65), (131, 77), (300, 301)):
        u = make('normal', rows, cols, 5).cuda()
        buf = torch.full((rows * cols + 128,), 3.0, device='cuda')
        need = ops.orthogonalize_workspace(u).numel()
        ws = torch.full((need + 4096,), 0x55, device='cuda', dtype=torch.uint8)
        o = ops.orthogonalize(u, out=buf[64:64 + rows * cols].view(rows, cols), workspace=ws)
        assert torch.equal(o, ops.orthogonalize(u))        # (a workspace full of other data gives the same bits)
        assert (buf[:64] == 3).all() and (buf[64 + rows * cols:] == 3).all() and (ws[need:] == 0x55).all()


def reference_update(p, g, m, fix, lr, mu, nesterov, wd, gs, steps, fold=True):
    p, g, m = p.double(), g.double(), m.double()
    if fix is not None and fold:
        f = {k: v.double().cpu() for k, v in fix.items()}
        g = f['scale'] * g - f['scale'] / f['sigma'] * f['dot'] * f['dsigma'].view(g.shape)
    g = gs * g
    m = mu * m + g
    u = g + mu * m if nesterov else m
    mat = u.reshape(-1, u.shape[-1])
    o = orth64(mat, steps).reshape(u.shape)
    c = lr * 0.2 * math.sqrt(max(mat.shape))
    return (1 - lr * wd) * p - c * o, m, c * tolerance(mat, o, steps), mat


@pytest.mark.parametrize('nesterov,wd,gs,sn', [(True, 0.0, 1.0, False), (False, 0.1, 0.25, False), (True, 0.01, 1.0, True), (False, 0.0, 0.5, True)])
def test_update_matches_the_formula(ops, nesterov, wd, gs, sn):
    shapes = [(3, 3, 3, 16), (4, 4, 16, 32), (3, 3, 48, 130), (200, 16), (7, 9)]
    lr, mu, steps = 0.02, 0.9, 5
    g = torch.Generator().manual_seed(11)
    ps, gs_, ms = ([torch.randn(*s, generator=g) * k for s in shapes] for k in (0.05, 1e-3, 1e-3))
    fixes = None
    if sn:
        fixes = []
        for s, w, gr in zip(shapes, ps, gs_):
            n = int(np.prod(s))
            fixes.append({k: v.cuda() for k, v in dict(dsigma=torch.randn(n, generator=g) / math.sqrt(n), dot=(w * gr).sum().reshape(1),
                                                       sigma=torch.tensor([1.7]), scale=torch.tensor([0.8])).items()})
    dev = lambda ts: [t.cuda() for t in ts]
    p1, g1, m1 = dev(ps), dev(gs_), dev(ms)
    po, mo = [torch.zeros_like(t) for t in p1], [torch.zeros_like(t) for t in p1]
    group = ops.MuonGroup(p1, g1, m1, fixups=fixes, out_params=po, out_momenta=mo)
    group.step(lr, momentum=mu, nesterov=nesterov, weight_decay=wd, grad_scale=gs, steps=steps)
    for i, s in enumerate(shapes):
        fx = fixes[i] if sn else None
        rp, rm, tol, mat = reference_update(ps[i], gs_[i], ms[i], fx, lr, mu, nesterov, wd, gs, steps)
        # momentum: the fix-up's and the sum's roundings, each 2^-24 of its terms
        terms = mu * ms[i].double().abs() + 3 * gs * gs_[i].double().abs() + (4 * gs * (fx['scale'] / fx['sigma'] * fx['dot'] * fx['dsigma']).double().abs().cpu().view(s) if sn else 0)
        assert ((mo[i].cpu().double() - rm).abs() <= 2.0 ** -24 * (4 * terms + rm.abs())).all()
        # parameter: the result's share (the roundings of U add to X0's), and two roundings of p
        err = float((po[i].cpu().double() - rp).norm())
        assert err <= 2 * tol + 2.0 ** -23 * float(ps[i].double().norm() + rp.norm()), (s, err, tol)
        assert torch.equal(p1[i].cpu(), ps[i]) and torch.equal(m1[i].cpu(), ms[i])           # out of place: inputs kept
    inplace = ops.MuonGroup(p1, g1, m1, fixups=fixes)
    inplace.step(lr, momentum=mu, nesterov=nesterov, weight_decay=wd, grad_scale=gs, steps=steps)
    assert all(torch.equal(a, b) for a, b in zip(p1 + m1, po + mo))
    if sn:                                                 # a caller that applied the fix-up itself: the plain read
        q, n = dev(ps), dev(ms)
        plain = ops.MuonGroup(q, g1, n, fixups=fixes)
        plain.fold_fixup = False
        plain.step(lr, momentum=mu, nesterov=nesterov, weight_decay=wd, grad_scale=gs)
        q2, n2 = dev(ps), dev(ms)
        ops.MuonGroup(q2, g1, n2).step(lr, momentum=mu, nesterov=nesterov, weight_decay=wd, grad_scale=gs)
        assert all(torch.equal(a, b) for a, b in zip(q + n, q2 + n2))


def test_many_updates_stay_with_the_reference(ops):
    """ten updates in place: momentum and parameters follow the 64-bit recursion"""
    g = torch.Generator().manual_seed(17)
    shape, lr, mu = (90, 150), 0.01, 0.95
    p, m = torch.randn(*shape, generator=g), torch.zeros(*shape)
    pd, gd, md = p.cuda(), torch.zeros(*shape, device='cuda'), m.cuda()
    group = ops.MuonGroup([pd], [gd], [md])
    rp, rm, tol = p.double(), m.double(), 0.0
    for _ in range(10):
        gr = torch.randn(*shape, generator=g)
        gd.copy_(gr)
        group.step(lr, momentum=mu, weight_decay=0.1)
        rp, rm, t, _ = reference_update(rp, gr, rm, None, lr, mu, True, 0.1, 1.0, 5)
        tol += 2 * t + 2.0 ** -23 * float(rp.norm())
    assert float((pd.cpu().double() - rp).norm()) <= tol and float((md.cpu().double() - rm).norm()) <= 40 * 2.0 ** -24 * float(rm.norm())


def test_streams_graphs_and_plans(ops):
    import ctypes
    from mmdgan_hip import _lib
    shapes = [(27, 16), (300, 130), (64, 64), (128, 40)]
    us = [make('normal', r, c, i).cuda() for i, (r, c) in enumerate(shapes)]
    want = ops.orthogonalize(us)
    outs = [torch.zeros_like(u) for u in us]
    ws = ops.orthogonalize_workspace(us)
    call = lambda: ops.orthogonalize(us, out=outs, workspace=ws)

    def same():
        torch.cuda.synchronize()
        ok = all(torch.equal(a, b) for a, b in zip(outs, want))
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        return ok
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    assert same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    same()
    for _ in range(3):
        graph.replay()
        assert same()
        ops.orthogonalize(us[::-1])
    lib = _lib.load()
    handle = ops.Handle(workspace_bytes=0)
    with handle:
        ops.check(lib.mmdgan_plan_begin(), 'plan_begin')
        call()
        pid = ctypes.c_int(-1)
        ops.check(lib.mmdgan_plan_end(ctypes.byref(pid)), 'plan_end')
        assert same()
        for _ in range(2):
            ops.check(lib.mmdgan_plan_replay(pid.value, -1), 'plan_replay')
            assert same()
        assert all(k[0].startswith('mu_') for k in ops.plan_kernels(pid.value))
    # two calls at once on two streams, a workspace each
    ws2, outs2 = ops.orthogonalize_workspace(us), [torch.zeros_like(u) for u in us]
    s2 = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s):
            call()
        with torch.cuda.stream(s2):
            ops.orthogonalize(us, out=outs2, workspace=ws2)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs2, want)) and same()


def test_refusals_on_the_device(ops):
    u = torch.randn(20, 30, device='cuda')
    with pytest.raises(ValueError, match='no matrix'):
        ops.orthogonalize(torch.randn(5, device='cuda'))
    for steps in (0, -1, 17):
        with pytest.raises(ValueError):
            ops.orthogonalize(u, steps=steps)
    with pytest.raises(ValueError):
        ops.orthogonalize(torch.empty(0, 4, device='cuda'))
    with pytest.raises(AssertionError):
        ops.orthogonalize(u.t())
    with pytest.raises(AssertionError):
        ops.orthogonalize(u.half())
    with pytest.raises(AssertionError):
        ops.orthogonalize(u, out=torch.empty(30, 20, device='cuda'))
    with pytest.raises(AssertionError, match='workspace'):
        ops.orthogonalize(u, workspace=torch.empty(64, device='cuda', dtype=torch.uint8))
    with pytest.raises(AssertionError):
        ops.MuonGroup([u], [u.t().contiguous()], [u.clone()])
    with pytest.raises(AssertionError):
        ops.MuonGroup([], [], [])


def test_workspaces_are_real_memory_and_outputs_apart(ops):
    """an expanded tensor counts more bytes than it has; a parameter given twice would be updated by two workgroups at once"""
    u, v = torch.randn(20, 30, device='cuda'), torch.randn(20, 30, device='cuda')
    fake = torch.zeros(1, device='cuda', dtype=torch.uint8).expand(1 << 24)
    with pytest.raises(AssertionError, match='workspace'):
        ops.orthogonalize(u, workspace=fake)
    g = ops.MuonGroup([u], [v], [torch.zeros_like(u)])
    with pytest.raises(AssertionError, match='workspace'):
        g.step(0.1, workspace=fake)
    for call in (lambda: ops.orthogonalize([u, v], out=[v, u]), lambda: ops.orthogonalize([u, v], out=[u, u]),
                 lambda: ops.MuonGroup([u, u], [v, v], [torch.zeros_like(u) for _ in range(2)]).step(0.1),
                 lambda: ops.MuonGroup([u], [v], [v]).step(0.1)):
        with pytest.raises(ValueError, match='overlaps'):
            call()
    a, b = ops.orthogonalize([u, u])                         # the same input twice is no conflict
    assert torch.equal(a, b)


@pytest.mark.parametrize('shapes', [[(65 + i, 90 - i) for i in range(20)], [(900, 1300), (1024, 1200), (1281, 901), (300, 3000), (1000, 1100), (513, 2049)] * 2])
def test_what_a_matrix_gets_does_not_depend_on_the_others(ops, shapes):
    """more large matrices than a launch's table holds; enough of them for the larger tiles of the last product.  Every element is the
    same sum in the same order: the bits of a call of its own"""
    us = [make('gradient', r, c, i).cuda() for i, (r, c) in enumerate(shapes)]
    together = ops.orthogonalize(us)
    for u, o in zip(us, together):
        assert torch.equal(ops.orthogonalize(u), o), u.shape
    ref = orth64(us[1].cpu())
    assert float((together[1].cpu().double() - ref).norm()) <= tolerance(us[1].cpu(), ref)
    ps, ms = [torch.randn_like(u) for u in us], [torch.zeros_like(u) for u in us]
    alone = [p.clone() for p in ps]
    for p, u in zip(alone, us):
        ops.MuonGroup([p], [u], [torch.zeros_like(u)]).step(0.1)
    ops.MuonGroup(ps, us, ms).step(0.1)
    assert all(torch.equal(p, q) for p, q in zip(ps, alone))


def test_a_captured_update_advances_like_eager_ones(ops):
    """momentum and parameters after replays of one captured update, eager work and synchronisations between them, are those of as many
    eager updates, bit for bit; unaligned tensors and a second group on another stream beside it"""
    shapes, g = [(27, 16), (300, 130), (64, 70), (129, 40), (70, 200)], torch.Generator().manual_seed(5)
    host = [[torch.randn(*s, generator=g) * k for s in shapes] for k in (0.05, 1e-3, 1e-3)]

    def odd(t):                                              # four bytes off a 16-byte boundary
        f = torch.zeros(t.numel() + 1, device='cuda')
        v = f[1:].view(t.shape)
        v.copy_(t)
        return v
    eager, graphed, other = ([[f(t) for t in ts] for ts in host] for f in (lambda t: t.cuda(), lambda t: t.cuda(), odd))
    groups = [ops.MuonGroup(*ts) for ts in (eager, graphed, other)]
    groups[1].step(0.0, momentum=1.0, grad_scale=0.0)        # (allocates its workspace; moves nothing)
    assert all(torch.equal(a, b) for a, b in zip(graphed[0] + graphed[2], eager[0] + eager[2]))
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        groups[1].step(0.02, momentum=0.9, weight_decay=0.01)
    torch.cuda.synchronize()
    for n in range(4):
        groups[0].step(0.02, momentum=0.9, weight_decay=0.01)
        if n % 2:
            torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(s):
            groups[2].step(0.02, momentum=0.9, weight_decay=0.01)
        torch.cuda.synchronize()
        for a, b, c in zip(eager[0] + eager[2], graphed[0] + graphed[2], other[0] + other[2]):
            assert torch.equal(a, b), n
            # (unaligned: the norm's sum in another order, its last bit in 64; that may flip roundings of X to 22 bits, 2^-22 of O's
            # entries before products that keep them, times a step of at most 0.02 * 0.2 * sqrt(300) = 0.07: far below 2^-20 of 0.2)
            assert float((a - c).abs().max()) <= 2.0 ** -20 * float(a.abs().max()), n
