"""How near the orthogonal factor is to the exact iterate, against measures that know nothing of the kernels' order of products: the same iteration on
32-bit products, and the rounding of the result's type.

fp32: an operand here is a value rounded to 32 bits (2^-24) and then to an fp16 pair (2^-23 at most), and a product leaves out lo * lo, of the size of
one rounding more: u^2 (1 + 4 + 1) against the 32-bit iteration's u^2, a factor of 2.5 on independent roundings.  The errors lie in few singular
directions, so a norm is a draw of few normal variables; over four matrices two such draws differ by less than 1.6 (chi-square of 4 against 4 at
2.5 / 97.5 %: 3.1 = 1.76^2 each way, and more than one direction a matrix carries the error): 4 in all.
16 bits: rounding alone is at rms r from the exact iterate; the kernels may add 3/4 of it: sqrt(1 + 9/16) = 1.25."""
import pytest
import torch

from tests.test_orthogonalise_gpu import exact
from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops

pytestmark = pytest.mark.gpu
A, B, C = ops.NS_COEFFICIENTS


def in_32_bits(x, steps=5):
    y = x.float()
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.mT.contiguous()
    y = (y.double() / (y.double().square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)).float()
    for _ in range(steps):
        g = torch.bmm(y, y.mT.contiguous())
        y = A * y + torch.bmm(B * g + C * torch.bmm(g, g), y)
    return y.mT if tall else y


def matrices(dev, m, n, kind, seed=3, batch=4):
    """directions:noise — a few directions of unit scale in noise."""
    r, noise = kind
    gen = torch.Generator(device=dev).manual_seed(seed)
    u, v = torch.randn(batch, m, r, generator=gen, device=dev), torch.randn(batch, r, n, generator=gen, device=dev)
    return torch.bmm(u, v) + noise * torch.randn(batch, m, n, generator=gen, device=dev)


SIZES = pytest.mark.parametrize('m, n', [(48, 600), (128, 512), (200, 200), (512, 512), (600, 1500), (1500, 600), (1024, 1024)])
KINDS = pytest.mark.parametrize('kind', [(1, 1e-1), (1, 1e-2), (1, 1e-3), (1, 1e-4), (8, 0.5), (8, 1e-2)], ids=lambda k: '%d:%g' % k)


@SIZES
@KINDS
def test_fp32_against_32_bit_products(dev, m, n, kind):
    x = matrices(dev, m, n, kind)
    want = exact(x)
    base = float((in_32_bits(x).double() - want).norm())
    for joined in (None, 1, 3):
        err = float((ops.orthogonalise(x, joined=joined).double() - want).norm())
        assert err <= 4 * base + 2.0 ** -24 * float(want.norm()), (joined, err / base)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'f16'])
@SIZES
@KINDS
def test_16_bits_against_their_rounding(dev, dtype, m, n, kind):
    x = matrices(dev, m, n, kind).to(dtype)
    want = exact(x)
    base = float((want.to(dtype).double() - want).norm())
    for joined in (None, 1, 3):
        err = float((ops.orthogonalise(x, joined=joined).double() - want).norm())
        assert err <= 1.25 * base, (joined, err / base)


@pytest.mark.parametrize('dtype, most', [(torch.float32, 1), (torch.float16, 3), (torch.bfloat16, 5)], ids=['f32', 'f16', 'bf16'])
def test_which_iterations_are_joined(dev, dtype, most):
    """None: by the type; single ones for nearly square matrices of over 128 rows, all of the call."""
    def same(x, joined, **k):
        got, want = ops.orthogonalise(x, **k), ops.orthogonalise(x, joined=joined, **k)
        return all(torch.equal(a, b) for a, b in (zip(got, want) if isinstance(x, list) else [(got, want)]))
    gen = torch.Generator(device=dev).manual_seed(1)
    x = [torch.randn(m, n, generator=gen, device=dev).to(dtype) for m, n in [(160, 170), (170, 160), (300, 300), (160, 171), (128, 128)]]
    for t in x[:3] + [x[:3]]:
        assert same(t, 1)
    for t in x[3:] + [x]:
        assert same(t, most)
    w, g = x[2].float().to(dtype), x[2].clone()
    plans = [w.clone(), w.clone()]
    for p, joined in zip(plans, (None, 1)):
        ops.muon_step([p], [g], [torch.zeros_like(w, dtype=torch.float32)], 0.1, joined=joined)
    assert torch.equal(*plans)


def test_joined_refusals(dev):
    x = torch.randn(8, 9, device=dev)
    for bad in (0, 17, -1):
        with pytest.raises(L.WgsError, match='joined must be'):
            ops.orthogonalise(x, joined=bad)
        with pytest.raises(L.WgsError, match='joined must be'):
            ops.muon_step([x], [x.clone()], [torch.zeros_like(x)], 0.1, joined=bad)
