"""Refusals of the group-norm entries: decided on the host, no device needed (pointers are never followed)."""
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
                     (dict(x=None), 'null'), (dict(stats=None), 'null'), (dict(ws=None), 'null')):
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
