"""When the library is built again: a change of a source, of a header or of the compiler's flags, and every time the driver entry asks."""
import importlib.util
import os
import stat
import sys

import pytest

from conftest import PKG, ROOT

FAKE = '''#!%s
import sys
out = sys.argv[sys.argv.index('-o') + 1]
open(out, 'w').write(' '.join(sys.argv[1:]))
open(%r, 'a').write(out + '\\n')
'''


@pytest.fixture
def ext(tmp_path):
    spec = importlib.util.spec_from_file_location('_build_ext_under_test', os.path.join(PKG, 'build_ext.py'))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.HERE, mod.CSRC, mod.OBJ, mod.LIB = (str(tmp_path / p) for p in ('pkg', 'pkg/csrc', 'pkg/build', 'pkg/lib/libx.so'))
    os.makedirs(mod.CSRC)
    os.makedirs(str(tmp_path / 'include'))
    (tmp_path / 'include' / 'mmdgan_hip.h').write_text('')
    for n in ('a', 'b'):
        (tmp_path / 'pkg' / 'csrc' / (n + '.hip')).write_text('')
    log = tmp_path / 'log'
    hipcc = tmp_path / 'hipcc'
    hipcc.write_text(FAKE % (sys.executable, str(log)))
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    mod.HIPCC = str(hipcc)

    def built():
        names = sorted(os.path.basename(p) for p in log.read_text().split()) if log.exists() else []
        log.write_text('')
        return names
    mod.built = built
    return mod


def test_rebuilds_what_changed(ext):
    ext.build(verbose=False)
    assert ext.built() == ['a.o', 'b.o', 'libx.so']
    ext.build(verbose=False)
    assert ext.built() == []
    os.utime(os.path.join(ext.CSRC, 'a.hip'), (2e9, 2e9))
    ext.build(verbose=False)
    assert ext.built() == ['a.o', 'libx.so']
    os.utime(os.path.join(ext.CSRC, 'a.hip'), (1e9, 1e9))
    ext.build(force=True, verbose=False)
    assert ext.built() == ['a.o', 'b.o', 'libx.so']


def test_objects_of_other_flags_are_built_again(ext):
    """objects left by a build with other flags (they are not in git, and outlive a change of the flags) must not be linked"""
    ext.build(verbose=False)
    ext.built()
    ext.FLAGS = ext.FLAGS + ['-DX']
    ext.build(verbose=False)
    assert ext.built() == ['a.o', 'b.o', 'libx.so']
    assert '-DX' in open(os.path.join(ext.OBJ, 'a.o')).read()
    ext.build(verbose=False)
    assert ext.built() == []


def test_the_driver_entry_compiles_every_time(monkeypatch):
    sys.path.insert(0, ROOT)
    import __graft_entry__ as g
    import build_ext
    calls = []
    monkeypatch.setattr(build_ext, 'build', lambda force=False, verbose=True: calls.append(force) or build_ext.LIB)
    g.build()
    assert calls == [True]


def test_no_device_code_is_compiled_with_packed_fp32():
    """every compiler line for gfx950 that names a .hip source carries the flag, the tools' too, and none writes packed fp32 by hand"""
    import glob
    import re
    flag, found = '-packed-fp32-ops', 0
    files = [f for p in ('tools/*', 'mmd-gan_amd/*.py', 'oracle/*.py', '*.py') for f in glob.glob(os.path.join(ROOT, p)) if os.path.isfile(f)]
    for f in files:
        if not f.endswith(('.sh', '.py', '.hip', '.md')):
            continue
        pieces = re.split(r'--offload-arch=gfx950', open(f).read())
        for piece in pieces[1:]:
            if re.search(r'\.hip\b', piece[:600].split('\n\n')[0]):
                found += 1
                assert flag in piece[:600], (f, piece[:200])
    assert found >= 14
    import build_ext
    assert flag in build_ext.FLAGS
    for f in glob.glob(os.path.join(ROOT, 'tools', '*.hip')) + glob.glob(os.path.join(ROOT, 'mmd-gan_amd', 'csrc', '*')):
        text = re.sub(r'//[^\n]*', '', open(f).read())
        assert not re.search(r'v_pk_(add|mul|fma)_f32', text), f
