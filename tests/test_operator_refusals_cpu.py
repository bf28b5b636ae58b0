"""CPU: what the operators of the training step refuse, through Python and through the C ABI (every check is on the host, before a launch)."""
import ctypes

import pytest
import torch

from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops

I64, F = ctypes.c_int64, ctypes.c_float
P = ctypes.c_void_p(4096)        # never dereferenced: the call is refused first


def refused(rc, text):
    assert rc != 0 and text in L.lib().wgs_last_error(), L.lib().wgs_last_error()


def test_label_logprobs_refuses_cpu_tensors():
    with pytest.raises(L.WgsError, match='no CPU fallback'):
        ops.label_logprobs(torch.randn(2, 8), torch.zeros(2, dtype=torch.int64))


def lp_fwd(logits=P, dtype=0, rows=4, V=5000, stride=5000, labels=P, top=2, logp=P, ws=P, ws_bytes=1 << 30, top_logp=P):
    return L.lib().wgs_label_logprobs_fwd(logits, dtype, I64(rows), I64(V), I64(stride), labels, I64(-100), top, logp, P, P, top_logp, P, ws,
                                          I64(ws_bytes), None)


def test_label_logprobs_forward_refusals():
    refused(lp_fwd(dtype=3), b'unknown dtype')
    refused(lp_fwd(V=0), b'bad sizes')
    refused(lp_fwd(V=1 << 30, stride=1 << 30), b'bad sizes')
    refused(lp_fwd(rows=-1), b'bad sizes')
    refused(lp_fwd(rows=1 << 24), b'bad sizes')
    refused(lp_fwd(stride=4999), b'bad sizes')
    refused(lp_fwd(top=65), b'top must be')
    refused(lp_fwd(top=-1), b'top must be')
    refused(lp_fwd(V=3, stride=3, top=4), b'top must be')
    refused(lp_fwd(logits=None), b'null pointer')
    refused(lp_fwd(labels=None), b'null pointer')
    refused(lp_fwd(top_logp=None), b'null pointer')
    refused(lp_fwd(logits=ctypes.c_void_p(4097), dtype=1), b'not aligned')
    need = L.lib().wgs_label_logprobs_ws_bytes(I64(4), I64(131072), 20)
    assert need > 0
    refused(lp_fwd(V=131072, stride=131072, top=20, ws_bytes=need - 1), b'workspace')
    refused(lp_fwd(V=131072, stride=131072, top=20, ws=None), b'workspace')
    assert lp_fwd(rows=0) == 0


def test_label_logprobs_backward_refusals():
    def bwd(dtype=1, rows=4, V=100, stride=100, gstride=100, grad=P, g_top=None, top=0, top_index=None):
        return L.lib().wgs_label_logprobs_bwd(P, dtype, I64(rows), I64(V), I64(stride), P, I64(-100), P, P, top, top_index, P, P, g_top, grad,
                                              I64(gstride), None)
    refused(bwd(dtype=-1), b'unknown dtype')
    refused(bwd(stride=99), b'bad sizes')
    refused(bwd(gstride=99), b'bad sizes')
    refused(bwd(grad=None), b'null pointer')
    refused(bwd(top=2, g_top=P), b'null pointer')
    refused(bwd(top=101), b'top must be')
    refused(bwd(grad=ctypes.c_void_p(4099)), b'not aligned')
    refused(bwd(rows=1 << 23, V=1 << 29, stride=1 << 29, gstride=1 << 29), b'too many scores')
    assert bwd(rows=0) == 0


def matrix(rows=8, cols=8, batch=1, ptr=4096, rs=8, mom=4096, bs=64, obs=64):
    return ops._MATRIX.pack(ptr, ptr, mom, bs, obs, rs, rs, rows, cols, batch, 0.1, 1.0, 0)


def ortho(*mats, dtype=0, steps=5, coef=ops.NS_COEFFICIENTS, eps=1e-7, ws=P, ws_bytes=1 << 40, step=False, mu=0.9):
    buf = ctypes.create_string_buffer(b''.join(mats) or b'\0')
    tail = [int(steps)] + [F(c) for c in coef] + [F(eps), ws, I64(ws_bytes), None]
    if step:
        return L.lib().wgs_muon_step(buf, len(mats), dtype, F(mu), 1, F(1.0), *tail)
    return L.lib().wgs_orthogonalise(buf, len(mats), dtype, *tail)


@pytest.mark.parametrize('step', [False, True])
def test_matrix_operators_refusals(step):
    refused(ortho(matrix(), dtype=5, step=step), b'unknown dtype')
    refused(ortho(matrix(), steps=0, step=step), b'steps')
    refused(ortho(matrix(), steps=17, step=step), b'steps')
    refused(ortho(matrix(rows=0), step=step), b'bad sizes')
    refused(ortho(matrix(rows=1 << 15, cols=1 << 15, rs=1 << 15), step=step), b'bad sizes')
    refused(ortho(matrix(rs=7), step=step), b'row strides')
    refused(ortho(matrix(batch=2, obs=63), step=step), b'batch strides')
    refused(ortho(matrix(batch=2, bs=-1), step=step), b'batch strides')
    refused(ortho(matrix(ptr=0), step=step), b'null pointer')
    refused(ortho(matrix(ptr=4098), step=step), b'not aligned')
    refused(ortho(matrix(), eps=-1.0, step=step), b'eps')
    refused(ortho(matrix(), eps=float('nan'), step=step), b'eps')
    refused(ortho(matrix(), coef=(40.0, 2.0, 1.0), step=step), b'bounded')
    refused(ortho(matrix(), coef=(float('nan'), 0.0, 0.0), step=step), b'bounded')
    refused(ortho(matrix(), coef=(0.0, 0.0, 0.0), step=step), b'bounded')
    refused(ortho(matrix(), ws=None, step=step), b'workspace')
    refused(ortho(matrix(), ws_bytes=16, step=step), b'workspace')
    refused(ortho(matrix(), ws=ctypes.c_void_p(4096 + 16), step=step), b'workspace')
    assert ortho(step=step) == 0 and ortho(matrix(batch=0), step=step) == 0
    if step:
        refused(ortho(matrix(mom=0), step=True), b'null pointer')
        refused(ortho(matrix(), step=True, mu=1.0), b'momentum')
        refused(ortho(matrix(), step=True, mu=float('nan')), b'momentum')


def test_workspace_of_a_list_is_that_of_its_largest_run():
    """Matrices go through in runs of a bounded workspace: a batch of any length needs no more than 4 GiB and one matrix."""
    lib = L.lib()
    one = lib.wgs_orthogonalise_ws_bytes(matrix(4096, 4096, 1, rs=4096, bs=1 << 24, obs=1 << 24), 1, 0, 5)
    many = lib.wgs_orthogonalise_ws_bytes(matrix(4096, 4096, 500, rs=4096, bs=1 << 24, obs=1 << 24), 1, 0, 5)
    assert 0 < one < many < (4 << 30) + one + (64 << 20)


def test_python_refuses_cpu_tensors():
    x = torch.randn(4, 4)
    with pytest.raises(L.WgsError, match='no CPU fallback'):
        ops.orthogonalise(x)
    with pytest.raises(L.WgsError, match='no CPU fallback'):
        ops.muon_step([x], [x], [x], 0.1)
    assert ops.orthogonalise([]) == [] and ops.muon_step([], [], [], 0.1) is None


def test_matrix_struct_matches_the_header(tmp_path):
    import os
    import re
    import subprocess
    hdr = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include')
    body = re.search(r'typedef struct wgs_matrix \{(.*?)\} wgs_matrix;', open(os.path.join(hdr, 'wgs.h')).read(), re.S).group(1)
    names = [re.search(r'(\w+)\s*$', piece).group(1) for decl in body.split(';') if decl.strip() for piece in decl.split(',')]
    src = tmp_path / 'm.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "wgs.h"\nint main(void) { printf("%zu", sizeof(wgs_matrix));'
                   + ''.join('printf(" %%zu", offsetof(wgs_matrix, %s));' % n for n in names) + 'return 0; }')
    exe = str(tmp_path / 'm')
    subprocess.run(['gcc', '-I', hdr, str(src), '-o', exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    import struct
    fmt = '3Q4q3i2fi'
    kinds = [c for n, c in re.findall(r'(\d*)(\D)', fmt) for _ in range(int(n or 1))]
    assert got[0] == ops._MATRIX.size and got[1:] == [struct.calcsize('=' + ''.join(kinds[:i])) for i in range(len(kinds))]
    assert ops._STEP_DECAY_AT == got[1 + names.index('step')]


def test_bucket_puts_the_orthogonalised_weights_first():
    from torch import nn
    from warpedganspace_amd.trainer import FlatBucket
    lin, conv, bn = nn.Linear(5, 3), nn.Conv2d(3, 4, 3), nn.BatchNorm2d(4)
    params = [lin.weight, bn.weight, conv.weight, conv.bias]
    want = conv.weight.detach().clone()
    b = FlatBucket([(1e-3, params), (1e-4, [lin.bias])], torch.device('cpu'), muon=True)
    assert b.segments[0][0] is conv.weight and b.muon_end == 108 and [n for _, _, n in b.segments] == [108, 15, 4, 4, 3]
    assert b.groups[0][1] == 0 and b.groups[0][2] == b.groups[1][1]
    assert torch.equal(conv.weight, want) and torch.equal(b.flat[:108].view(4, 3, 3, 3).permute(0, 3, 1, 2), want)
    plain = FlatBucket([(1e-3, [nn.Linear(2, 2).weight])], torch.device('cpu'))
    assert plain.muon_end == 0


def test_command_line():
    import train
    a = train.parse(['--gan-type', 'StyleGAN2', '--optimizer', 'muon', '--lambda-ent', '0.1', '--label-top', '5'])
    assert (a.optimizer, a.lambda_ent, a.label_top) == ('muon', 0.1, 5)
    d = train.parse(['--gan-type', 'StyleGAN2'])
    assert (d.optimizer, d.lambda_ent, d.label_top) == ('adam', 0.0, 0)
