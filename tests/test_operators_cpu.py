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
