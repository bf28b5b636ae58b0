"""Forms of wgs_orthogonalise and wgs_muon_step that only the C interface has: results in place, momenta of a batch, one input for a whole batch, and
batches of over one run's 4 GiB of workspace.  Tolerances: those of the sizes' own tests."""
import ctypes

import pytest
import torch

from tests.test_orthogonalise_gpu import HALF, check, exact, matrices, noisy, phases_of, step_exact
from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops

pytestmark = pytest.mark.gpu
F = ctypes.c_float
DT = pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
# one launch; a launch a step (fp32) or the chain kernel's; the general path
SHAPES = pytest.mark.parametrize('shape', [(3, 33, 65), (5, 21, 7), (3, 63, 1001), (3, 97, 301), (2, 301, 257)], ids=str)


def call(entries, dtype, muon=None, steps=5):
    """entries: (in, out, momentum or None, in batch stride, step, decay); in / out [batch, M, N] with adjacent elements."""
    mats = b''.join(ops._MATRIX.pack(x.data_ptr(), o.data_ptr(), m.data_ptr() if m is not None else 0, bs, o.stride(0), x.stride(-2), o.stride(-2),
                                     o.shape[1], o.shape[2], o.shape[0], lr, decay, 0) for x, o, m, bs, lr, decay in entries)
    lib, code = L.lib(), ops._DTYPES[dtype]
    size = lib.wgs_muon_step_ws_bytes if muon else lib.wgs_orthogonalise_ws_bytes
    need = size(mats, len(entries), code, steps)
    ws = torch.empty(need, dtype=torch.uint8, device=entries[0][1].device)
    tail = [steps] + [F(c) for c in ops.NS_COEFFICIENTS] + [F(1e-7), L.rawptr(ws), L.c_int64(need), L.stream()]
    if muon:
        mu, nesterov, scale = muon
        L.check(lib.wgs_muon_step(mats, len(entries), code, F(mu), nesterov, F(scale), *tail))
    else:
        L.check(lib.wgs_orthogonalise(mats, len(entries), code, *tail))
    return need


@DT
@SHAPES
def test_in_place(dev, dtype, shape):
    x = matrices(dev, shape, dtype, 7)
    keep, out = x.clone(), torch.empty_like(x)
    call([(x, out, None, x.stride(0), 0.0, 0.0)], dtype)
    assert torch.equal(x, keep)
    check(out, keep)
    call([(x, x, None, x.stride(0), 0.0, 0.0)], dtype)
    assert torch.equal(x, out)
    wide = torch.full((shape[0], shape[1], shape[2] + 3), 7.0, dtype=dtype, device=dev)      # rows with something between them
    wide[..., 1:1 + shape[2]] = keep
    view = wide[..., 1:1 + shape[2]]
    call([(view, view, None, view.stride(0), 0.0, 0.0)], dtype)
    check(view, keep)
    assert (wide[..., 0] == 7).all() and (wide[..., 1 + shape[2]:] == 7).all()


def near(w, m, want, lr, dtype):
    w1, m1, u, f = want
    assert float((m.double() - m1).abs().max()) <= 3 * 2.0 ** -24 * float(m1.abs().max() + 5)
    model = (noisy(u.float(), phases_of(dtype, 5)) - exact(u.float())).square().sum().sqrt()
    allowed = lr * (12 * model + 2.0 ** -20 * exact(u).square().sum().sqrt()) + 1.1 * HALF[dtype] * w1.square().sum().sqrt()
    assert float((w.double() - w1).square().sum().sqrt()) <= float(allowed)


@DT
@SHAPES
@pytest.mark.parametrize('shared', [False, True], ids=['', 'one gradient'])
def test_momenta_of_a_batch(dev, dtype, shape, shared):
    """An odd number of elements an instance: momenta of the later ones begin off a 16-byte block."""
    w, g, m = matrices(dev, shape, dtype, 1) * 0.1, matrices(dev, shape, dtype, 2), matrices(dev, shape, torch.float32, 3)
    lr = 0.05
    want = [step_exact(w[i], g[0 if shared else i], m[i], lr, 0.9, True, 0.1, 0.5, scale=1.0) for i in range(shape[0])]
    call([(g, w, m, 0 if shared else g.stride(0), lr, 1 - lr * 0.1)], dtype, muon=(0.9, 1, 0.5))
    for i in range(shape[0]):
        near(w[i], m[i], want[i], lr, dtype)


def test_a_batch_of_more_than_one_run(dev):
    """130 x 1024 in fp32 takes some 2 MB of planes: 2300 of them pass 4 GiB, and the batch is cut."""
    n, M, N = 2300, 130, 1024
    one = torch.empty(1, M, N, device=dev)
    gen = torch.Generator(device=dev).manual_seed(5)
    m = torch.randn(n, M, N, generator=gen, device=dev)
    x = torch.randn(n, M, N, generator=gen, device=dev)
    first = call([(x[:1], one, None, 0, 0.0, 0.0)], torch.float32)
    at = (4 << 30) // first
    samples = [0, 1, n // 2] + list(range(at - 30, at + 31, 3)) + [n - 1]
    assert 1000 < at < n - 60
    out = torch.empty_like(x)
    need = call([(x, out, None, x.stride(0), 0.0, 0.0)], torch.float32)
    assert need < (4 << 30) + (64 << 20)
    check(out[samples], x[samples])
    assert not out.isnan().any()
    # out now serves as the weights, x[0] as every instance's gradient
    lr = 0.05
    keep_w, keep_m = out[samples].clone(), m[samples].clone()
    call([(x, out, m, 0, lr, 1.0)], torch.float32, muon=(0.9, 0, 1.0))
    for k, i in enumerate(samples):
        near(out[i], m[i], step_exact(keep_w[k], x[0], keep_m[k], lr, 0.9, False, 0.0, scale=1.0), lr, torch.float32)
    assert not out.isnan().any() and not m.isnan().any()
