"""CPU: how the HIP library is built."""
import glob
import os
import re

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
