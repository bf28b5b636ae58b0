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
