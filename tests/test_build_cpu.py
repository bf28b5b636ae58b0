"""CPU: how the HIP library is built."""
import glob
import os
import re
import shutil
import subprocess
import time

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'warpedganspace_amd', 'csrc')
SCRIPT = open(os.path.join(CSRC, 'build.sh')).read()


def test_no_packed_fp32_instructions():
    """Neither written by hand nor made by the compiler, in any source."""
    for f in glob.glob(os.path.join(CSRC, '*')):
        if os.path.isfile(f) and f.endswith(('.hip', '.h', '.inc')):
            assert not re.search(r'v_pk_(add|mul|fma)_f32', open(f).read()), f
    flags = re.search(r'^FLAGS="(.*)"$', SCRIPT, re.M).group(1)
    assert '-Xclang -target-feature -Xclang -packed-fp32-ops' in flags
    compiles = [ln for ln in SCRIPT.splitlines() if re.search(r'\$HIPCC.* -c ', ln)]
    assert compiles and all('$FLAGS' in ln for ln in compiles)


def _copy(tmp_path):
    """The sources beside a compiler that only leaves an empty output."""
    csrc = tmp_path / 'pkg' / 'csrc'
    csrc.mkdir(parents=True)
    (tmp_path / 'include').mkdir()
    for f in glob.glob(os.path.join(CSRC, '*')):
        if os.path.isfile(f):
            shutil.copy2(f, csrc)
    shutil.copy2(os.path.join(CSRC, '..', '..', 'include', 'wgs.h'), tmp_path / 'include')
    cc = tmp_path / 'cc'
    cc.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then : > "$2"; fi; shift; done\n')
    cc.chmod(0o755)
    return csrc, dict(os.environ, HIPCC=str(cc))


def test_a_change_of_the_flags_rebuilds_every_object(tmp_path, monkeypatch):
    from warpedganspace_amd import _lib as L
    csrc, env = _copy(tmp_path)
    monkeypatch.setattr(L, '_HERE', str(csrc.parent))
    monkeypatch.setattr(L, 'HEADER_PATH', str(tmp_path / 'include' / 'wgs.h'))
    monkeypatch.setattr(L, 'LIB_PATH', str(csrc.parent / 'libwgs_hip.so'))

    def build():
        out = subprocess.run(['bash', str(csrc / 'build.sh')], env=env, check=True, capture_output=True, text=True).stdout
        assert L.library_matches_sources() is True
        return out.count('[hipcc]')
    sources = len(glob.glob(str(csrc / '*.hip')))
    assert build() == sources
    assert build() == 0
    script = csrc / 'build.sh'
    script.write_text(script.read_text().replace('-O3', '-O2'))
    assert L.library_matches_sources() is False
    later = time.time() + 60
    os.utime(script, (later, later))
    assert build() == sources


def test_a_failed_compilation_ends_the_build(tmp_path):
    """Not linked from an older object: the next run compiles that source again."""
    csrc, env = _copy(tmp_path)
    run = ['bash', str(csrc / 'build.sh')]
    subprocess.run(run, env=env, check=True, capture_output=True)
    library = csrc.parent / 'libwgs_hip.so'
    library.unlink()
    later = time.time() + 60
    os.utime(csrc / 'core.hip', (later, later))
    cc = tmp_path / 'cc'
    good = cc.read_text()
    cc.write_text(good.replace('#!/bin/sh\n', '#!/bin/sh\ncase "$*" in *core.hip*) exit 1;; esac\n'))
    assert subprocess.run(run, env=env, capture_output=True).returncode != 0
    assert not library.exists() and not (csrc / 'build' / 'core.o').exists()
    cc.write_text(good)
    out = subprocess.run(run, env=env, check=True, capture_output=True, text=True).stdout
    assert out.count('[hipcc]') == 1 and library.exists()
