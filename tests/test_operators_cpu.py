"""Refusals of the group-norm and orthogonalised-update entries: decided on the host, no device needed (pointers are never followed)."""
import pytest

from mmdgan_hip import _lib


@pytest.fixture(scope='module')
def lib():
    return _lib.load()


def message(lib):
    return lib.mmdgan_last_error().decode()


def test_group_norm_refuses_bad_geometries(lib):
    def fwd(N=2, HW=9, C=12, G=3, eps=1e-5, act=0, x=16, stats=16, ws=16):
        return lib.mmdgan_gn_fwd(x, N, HW, C, G, 16, 16, eps, act, 16, stats, ws, None)
    for kw, word in ((dict(N=0), 'bad size'), (dict(HW=0), 'bad size'), (dict(C=0), 'bad size'), (dict(G=0), 'bad size'),
                     (dict(G=-1), 'bad size'), (dict(G=5), 'do not divide'), (dict(G=24), 'do not divide'), (dict(act=4), 'activation'),
                     (dict(act=-1), 'activation'), (dict(eps=0.0), 'eps'), (dict(N=65536), 'too large'), (dict(HW=1 << 30), 'too large'),
                     (dict(ws=24), 'aligned'), (dict(x=None), 'null'), (dict(stats=None), 'null'), (dict(ws=None), 'null')):
        assert fwd(**kw) == -1, kw
        assert word in message(lib), (kw, message(lib))

    def bwd(N=4, xb=4, HW=9, C=12, G=3, act=0, x=16, dx=32):
        return lib.mmdgan_gn_bwd(x, 48, N, xb, HW, C, G, 16, 16, 16, act, dx, None, None, 16, None)
    for kw, word in ((dict(xb=5), 'x_batch'), (dict(xb=1), 'x_batch'), (dict(xb=-1), 'x_batch'), (dict(G=7), 'do not divide'),
                     (dict(x=None), 'null'), (dict(dx=None), 'null'), (dict(xb=2, dx=16), 'dx must not be x')):
        assert bwd(**kw) == -1, kw
        assert word in message(lib), (kw, message(lib))
    assert lib.mmdgan_gn_workspace_bytes(2, 9, 12, 5) == 0 and lib.mmdgan_gn_workspace_bytes(0, 9, 12, 3) == 0
    assert lib.mmdgan_gn_workspace_bytes(2, 9, 12, 3) > 0


def test_orthogonalised_updates_refuse_bad_jobs(lib):
    import ctypes
    from mmdgan_hip.ops import MuonJob

    def job(rows=8, cols=8, **kw):
        j = (MuonJob * 1)()
        for f in ('grad', 'out', 'param', 'momentum', 'momentum_out'):
            setattr(j[0], f, kw.get(f, 16))
        for f in ('dsigma', 'dot', 'sigma', 'scale'):
            setattr(j[0], f, kw.get(f))
        j[0].rows, j[0].cols = rows, cols
        return ctypes.cast(j, ctypes.c_void_p), j

    def orth(n=1, steps=5, ws=16, **kw):
        p, keep = job(**kw)
        return lib.mmdgan_orthogonalize(p, n, steps, ws, None)

    def update(n=1, steps=5, ws=16, **kw):
        p, keep = job(**kw)
        return lib.mmdgan_muon_update(p, n, 0.1, 0.9, 1, 0.0, 1.0, 1, steps, ws, None)
    for call in (orth, update):
        for kw, word in ((dict(n=0), 'no matrices'), (dict(steps=0), 'steps'), (dict(steps=17), 'steps'), (dict(rows=0), 'side'),
                         (dict(cols=-3), 'side'), (dict(rows=8193, cols=8193), 'side'), (dict(rows=1, cols=(1 << 22) + 1), 'side'),
                         (dict(rows=1024, cols=1 << 21), 'side'), (dict(ws=None), 'workspace'), (dict(ws=24), 'workspace'),
                         (dict(grad=None), 'null'), (dict(out=None), 'null')):
            assert call(**kw) == -1, kw
            assert word in message(lib), (kw, message(lib))
    for kw, word in ((dict(param=None), 'null'), (dict(momentum=None), 'null'), (dict(momentum_out=None), 'null'),
                     (dict(dsigma=16), 'dsigma without'), (dict(dsigma=16, dot=16, sigma=16), 'dsigma without')):
        assert update(**kw) == -1, kw
        assert word in message(lib), (kw, message(lib))
    assert lib.mmdgan_orthogonalize(None, 1, 5, 16, None) == -1
    size = lambda steps=5, **kw: lib.mmdgan_muon_workspace_bytes(job(**kw)[0], 1, steps)
    assert size() > 0 and size(steps=0) == 0 and size(rows=0) == 0 and size(rows=9000, cols=9000) == 0


def test_group_norm_refuses_overlaps(lib):
    A, B, size = 1 << 20, 1 << 22, 4 * 9 * 12 * 4           # addresses that are only compared

    def fwd(y):
        return lib.mmdgan_gn_fwd(A, 4, 9, 12, 3, 16, 16, 1e-5, 0, y, 16, 16, None)

    def bwd(dx, xb=4, dgamma=None, dbeta=None):
        return lib.mmdgan_gn_bwd(A, B, 4, xb, 9, 12, 3, 16, 16, 16, 0, dx, dgamma, dbeta, 16, None)
    for call in (lambda: fwd(A + 16), lambda: fwd(A - size + 4), lambda: fwd(A + size - 4), lambda: bwd(A + 16), lambda: bwd(A - size + 4),
                 lambda: bwd(B + 16), lambda: bwd(B + size - 4), lambda: bwd(1 << 24, 4, 1 << 25, (1 << 25) + 44)):
        assert call() == -1 and 'overlap' in message(lib)
    assert bwd(A, xb=2) == -1 and 'dx must not be x' in message(lib)


def test_orthogonalised_updates_refuse_overlaps(lib):
    """an output may be its own matrix's input, and overlaps nothing else: another matrix reads it at a time that is not fixed"""
    import ctypes
    from mmdgan_hip.ops import MuonJob
    base, size = 1 << 20, 8 * 100 * 4                        # addresses that are only compared
    names = ('grad', 'out', 'param', 'momentum', 'momentum_out', 'dsigma')

    def jobs(*change):
        j = (MuonJob * 2)()
        for i in range(2):
            for k, f in enumerate(names):
                setattr(j[i], f, base + (i * 8 + k) * 4096)
            j[i].dot = j[i].sigma = j[i].scale = base - 64
            j[i].rows, j[i].cols = (8, 100) if i == 0 else (100, 8)
        for i, f, i2, f2, off in change:
            setattr(j[i], f, getattr(j[i2], f2) + off)
        return ctypes.cast(j, ctypes.c_void_p), j

    def orth(*change):
        p, keep = jobs(*change)
        return lib.mmdgan_orthogonalize(p, 2, 5, 16, None)

    def update(*change):
        p, keep = jobs(*change)
        return lib.mmdgan_muon_update(p, 2, 0.1, 0.9, 1, 0.0, 1.0, 1, 5, 16, None)
    for change in ((0, 'out', 1, 'grad', 0), (1, 'out', 0, 'grad', 0), (0, 'out', 1, 'out', 0), (0, 'out', 0, 'grad', 16),
                   (1, 'out', 1, 'grad', 4 - size), (1, 'out', 0, 'grad', size - 4)):
        assert orth(change) == -1 and 'overlaps' in message(lib), change
    for a in ('out', 'momentum_out'):
        for i in range(2):
            for k in range(2):
                for b in names:
                    own = i == k and (a, b) in (('out', 'param'), ('momentum_out', 'momentum'))
                    for off in (16, 4 - size) if own else () if i == k and a == b else (0, 16, size - 4):
                        assert update((i, a, k, b, off)) == -1 and 'overlaps' in message(lib), (i, a, k, b, off)


def test_tensors_of_another_device_are_refused(monkeypatch):
    """launches go to the current device: the check itself, with stand-ins for tensors"""
    import torch
    from mmdgan_hip import ops

    class T:
        def __init__(self, d):
            self.d = d

        def get_device(self):
            return self.d
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 1)
    ops._on_current_device(T(1), None, T(1))
    for bad in ((T(0),), (T(1), T(0)), (T(1), None, T(-1))):
        with pytest.raises(AssertionError, match='device'):
            ops._on_current_device(*bad)


def test_sides_that_do_not_fit_an_int_are_refused():
    import torch
    from mmdgan_hip import ops
    wide = torch.empty(1, device='meta').expand(1 << 33, 2)
    for t in (wide, wide.t()):
        with pytest.raises(ValueError, match='8589934592'):
            ops._muon_jobs([t])
    g = torch.empty(1, device='meta').expand((1 << 32) + 4)
    with pytest.raises(AssertionError, match='4294967300'):
        ops._gn_geometry(g[None], g, g, 4)


def test_group_norm_has_no_workspace_for_sizes_the_entries_refuse(lib):
    """0 bytes, as documented, for every size that the entries refuse - also for one whose chunk length does not fit an int (it divided by
    zero once)"""
    size = lib.mmdgan_gn_workspace_bytes
    for N, HW, C, G in ((65536, 9, 12, 3), (70000, 9, 12, 3), (2, 1 << 30, 12, 3), (1, 1 << 38, 4, 1), (1, 1 << 38, 1, 1), (1, (1 << 63) - 1, 1, 1),
                        (1, -5, 4, 1), (2, 0, 4, 1), (2, 9, 0, 1), (2, 9, 12, 0), (2, 9, 12, -3)):
        assert size(N, HW, C, G) == 0, (N, HW, C, G)
        assert lib.mmdgan_gn_fwd(16, N, HW, C, G, 16, 16, 1e-5, 0, 16, 16, 16, None) == -1
    assert size(65535, 9, 12, 3) > 0 and size(1, 0x7fffffff, 1, 1) > 0 and size(1, 0x7fffffff // 12, 12, 3) > 0
    from mmdgan_hip import ops
    for N, HW, C, G in ((65536, 9, 12, 3), (1, 1 << 38, 4, 1)):
        with pytest.raises(ValueError, match='group_norm'):
            ops.group_norm_workspace(N, HW, C, G, 'cpu')
