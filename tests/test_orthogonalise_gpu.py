"""Newton-Schulz orthogonalisation and the momentum step that applies it, against the iteration in 64 bits.

Tolerance: the kernels' error is a sum of independent roundings.  An operand of a product is an fp16 pair, off by at most 2^-22 of its value
(half a step of the low part; 16-bit inputs are exact); a product's sum of K terms is rounded to 24 bits at most 3 K / 16 times, each time off by
at most 2^-24 of a partial sum that is itself at most of the order of the root of the terms' squares.  So an entry of P R is off by a random
amount of about u sqrt((P o P) (R o R)), u = 2^-22 + 2^-24 sqrt(3 K / 16).  `noisy` runs the same order of products in 64 bits with exactly this
noise added to every product; the result's distance from the exact iterate is the expected error, and six times that (plus the rounding
of the output) is what is allowed in the Frobenius norm; `check` says what that allows the largest entry."""
import math

import pytest
import torch

from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
C3 = ops.NS_COEFFICIENTS


def exact(x, steps=5, coef=C3, eps=1e-7):
    a, b, c = coef
    y = x.double()
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.mT.contiguous()
    y = y / (y.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        g = y @ y.mT.contiguous()
        y = a * y + (b * g + c * g @ g) @ y
    return y.mT if tall else y


def noisy(x, phases, coef=C3, eps=1e-7, seed=0):
    """The kernels' order of products (phases of so many iterations) with the rounding of every product added at random."""
    a, b, c = coef
    gen = torch.Generator(device=x.device).manual_seed(seed)

    def mul(p, r):
        k = p.shape[-1]
        u = 2.0 ** -22 + 2.0 ** -24 * math.sqrt(3 * k / 16)
        out = p @ r
        return out + u * ((p * p) @ (r * r)).sqrt() * (2 * torch.rand(out.shape, generator=gen, dtype=out.dtype, device=out.device) - 1)
    y = x.double()
    if y.shape[-2] > y.shape[-1]:
        y = y.mT.contiguous()
    y = y / (y.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    eye = torch.eye(y.shape[-2], dtype=y.dtype, device=y.device)
    for n in phases:
        g = mul(y, y.mT.contiguous())
        q = None
        for i in range(n):
            w = a * eye + b * g + c * mul(g, g)
            q = w if q is None else mul(q, w)
            if i + 1 < n:
                g = mul(mul(w, g), w)
                g = (g + g.mT) / 2
        y = mul(q, y)
    return y.mT if x.shape[-2] > x.shape[-1] else y


def phases_of(dtype, steps, step=False):
    most = {torch.float32: 1, torch.float16: 3, torch.bfloat16: 5}[dtype]
    n = -(-steps // most)
    out, left = [], steps
    for i in range(n):
        out.append(-(-left // (n - i)))
        left -= out[-1]
    return out


def check(got, x, steps=5, coef=C3, eps=1e-7, dtype=None):
    dtype = dtype or x.dtype
    want = exact(x, steps, coef, eps)
    # After many steps the error lies in few singular directions, and along one the size of a single draw of the noise is a |normal| variable: under
    # a sixth of its scale once in 7.6 draws.  The root mean square of eight draws is not (P(chi2_8 / 8 < 1 / 36) < 1e-6).
    draws = 8 if steps > 5 else 1
    model = (sum((noisy(x, phases_of(dtype, steps), coef, eps, seed) - want).square().sum((-2, -1)) for seed in range(draws)) / draws).sqrt()
    size = want.square().sum((-2, -1)).sqrt()
    err = got.double() - want
    fro = err.square().sum((-2, -1)).sqrt()
    allowed = 6 * model + 1.1 * HALF[dtype] * size + 2.0 ** -24 * size + 1e-30
    assert (fro <= allowed).all(), (float((fro / allowed).max()), float((fro / size).max()), float((model / size).max()))
    count = x.shape[-2] * x.shape[-1]
    top = err.abs().amax((-2, -1))
    # The largest entry: an error E whose entries are independent has |E|_max of about |E|_F sqrt(2 ln(M N)) / sqrt(M N).  But after many steps E
    # lies in few singular directions (the map's derivative differs from one singular value to the next and multiplies up), and for one,
    # E = |E|_F u v^T with unit vectors whose largest entries are about sqrt(2 ln M / M) and sqrt(2 ln N / N): the product of the two is allowed.
    rms = 6 * model / math.sqrt(count) * math.sqrt((2 * math.log(x.shape[-2]) + 2) * (2 * math.log(x.shape[-1]) + 2)) + HALF[dtype] * want.abs().amax((-2, -1)) + 2.0 ** -24 * size
    assert (top <= rms + 1e-30).all(), (float((top / rms).max()),)


def matrices(dev, shape, dtype, seed, kind='noise'):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(shape, generator=gen, device=dev)
    if kind == 'spiked':
        u = torch.randn(shape[:-1] + (1,), generator=gen, device=dev)
        v = torch.randn(shape[:-2] + (1, shape[-1]), generator=gen, device=dev)
        x = 0.1 * x + u @ v
    elif kind == 'rank':
        r = max(1, min(shape[-2:]) // 3)
        x = torch.randn(shape[:-1] + (r,), generator=gen, device=dev) @ torch.randn(shape[:-2] + (r, shape[-1]), generator=gen, device=dev)
    elif kind == 'rows':
        x = x * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=gen, device=dev))
    return x.to(dtype)


DT = pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])


@DT
@pytest.mark.parametrize('shape', [(1, 1), (1, 7), (5, 1), (2, 3), (31, 33), (32, 32), (33, 31), (64, 576), (65, 64), (63, 200), (100, 2100), (129, 127), (257, 300), (300, 1000),
                                   (1000, 130), (512, 4608), (1, 5000), (640, 641)], ids=str)
def test_sizes(dev, dtype, shape):
    x = matrices(dev, shape, dtype, sum(shape))
    check(ops.orthogonalise(x), x)


@DT
@pytest.mark.parametrize('shape', [(1500, 1500), (2048, 700), (1100, 4100)], ids=str)
def test_large(dev, dtype, shape):
    x = matrices(dev, shape, dtype, sum(shape))
    check(ops.orthogonalise(x), x)


@DT
@pytest.mark.parametrize('kind', ['spiked', 'rank', 'rows'])
@pytest.mark.parametrize('shape', [(3, 96, 200), (2, 300, 256)], ids=str)
def test_spectra(dev, dtype, kind, shape):
    x = matrices(dev, shape, dtype, 5, kind)
    check(ops.orthogonalise(x), x)


@DT
@pytest.mark.parametrize('steps', [2, 3, 5, 8])
@pytest.mark.parametrize('shape', [(33, 4100), (2, 64, 2500), (66, 66), (3, 97, 101), (128, 128), (2, 300, 120)], ids=str)
def test_few_rows(dev, dtype, steps, shape):
    x = matrices(dev, shape, dtype, 3, 'rows')
    check(ops.orthogonalise(x, steps=steps), x, steps)


@DT
@pytest.mark.parametrize('shape', [(3, 64, 513), (64, 1100), (16, 33, 2048), (17, 33, 2017), (32, 897), (2, 2000, 20), (2, 640, 64), (1, 1537)], ids=str)
def test_short_matrices_with_many_columns(dev, dtype, shape):
    x = matrices(dev, shape, dtype, 11)
    check(ops.orthogonalise(x), x)


@pytest.mark.parametrize('shapes', [[(64, 900), (8, 30), (200, 3)], [(1200, 20), (32, 40), (1, 1)]], ids=str)
def test_short_steps_together(dev, shapes):
    """A long and some short matrices in the launches of one step: workgroups without columns leave."""
    ws, gs, ms = ([matrices(dev, s, torch.float32, 10 * k + i) for i, s in enumerate(shapes)] for k in range(3))
    want = [step_exact(w, g, m, 0.05, 0.9, True, 0.1, 0.5) for w, g, m in zip(ws, gs, ms)]
    ops.muon_step(ws, gs, ms, 0.05, momentum=0.9, nesterov=True, weight_decay=0.1, grad_scale=0.5)
    for w, m, (w1, m1, u, f) in zip(ws, ms, want):
        assert float((m.double() - m1).abs().max()) <= 3 * 2.0 ** -24 * float(m1.abs().max() + 5)
        model = (noisy(u.float(), phases_of(torch.float32, 5)) - exact(u.float())).square().sum().sqrt()
        allowed = 0.05 * f * (12 * model + 2.0 ** -20 * exact(u).square().sum().sqrt()) + 1.1 * 2.0 ** -24 * w1.square().sum().sqrt()
        assert float((w.double() - w1).square().sum().sqrt()) <= float(allowed)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'f16'])
@pytest.mark.parametrize('shapes', [[(33, 4100), (2, 128, 140), (1, 2500), (90, 3)], [(1, 4100), (31, 2100), (2, 64, 2049)], [(128, 300), (129, 300)]], ids=str)
def test_few_rows_together(dev, dtype, shapes):
    xs = [matrices(dev, s, dtype, i) for i, s in enumerate(shapes)]
    for got, x in zip(ops.orthogonalise(xs), xs):
        check(got, x)


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 6, 7, 11, 16])
@DT
def test_steps_and_coefficients(dev, dtype, steps):
    x = matrices(dev, (2, 70, 150), dtype, steps)
    check(ops.orthogonalise(x, steps=steps), x, steps)
    cubic = (1.5, -0.5, 0.0)
    check(ops.orthogonalise(x, steps=steps, coefficients=cubic), x, steps, cubic)


def test_singular_values_and_vectors(dev):
    x = matrices(dev, (200, 500), torch.float32, 9)
    o = ops.orthogonalise(x).double()
    s = torch.linalg.svdvals(o)
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25
    p = torch.linalg.svd(x.double(), full_matrices=False)
    core = p.U.T @ o @ p.Vh.T                                 # diagonal: the singular vectors are x's
    off = core - torch.diag(torch.diagonal(core))
    assert float(off.abs().max()) < 1e-4


@DT
@pytest.mark.parametrize('scale', [1e-30, 1e-20, 1e-6, 1.0, 1e4, 1e30])
def test_scales(dev, dtype, scale):
    """The result does not depend on the scale down to where eps counts; far below it is proportional to the input."""
    x = matrices(dev, (40, 90), torch.float32, 3) * scale
    if dtype == torch.float16 and not 1e-6 <= scale <= 1e4:
        pytest.skip('outside the type')
    x = x.to(dtype)
    got = ops.orthogonalise(x)
    assert torch.isfinite(got).all()
    want = exact(x)
    tiny = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -24
    assert float((got.double() - want).abs().max()) <= (2 * HALF[dtype] + 1e-3 * (dtype != torch.float32) + 3e-5) * float(want.abs().max()) + tiny
    z = ops.orthogonalise(x, eps=0.0)
    check(z, x, eps=0.0)


def test_zero_nan_and_infinity(dev):
    x = matrices(dev, (5, 50, 60), torch.float32, 1)
    x[1] = 0
    x[2, 3, 4] = math.nan
    x[3, 49, 59] = math.inf
    x[4] *= 1e38
    for eps in (1e-7, 0.0):
        o = ops.orthogonalise(x, eps=eps)
        assert (o[1] == 0).all() and o[2].isnan().all() and o[3].isnan().all()
        assert x[4].isinf().any() and o[4].isnan().all()      # (1e38 times a normal sample passes the type's range)
        check(o[:1], x[:1])


def test_largest_finite_values(dev):
    x = matrices(dev, (50, 60), torch.float32, 1) * 5e37
    assert x.isfinite().all() and float(x.abs().max()) > 1e38
    check(ops.orthogonalise(x), x)


@DT
def test_strides(dev, dtype):
    base = matrices(dev, (6, 80, 130), dtype, 2)
    for x in (base[::2], base[:, 3:70, 5:100], base.mT, base[:, ::2], base[:, :, ::3], base[0], base[0].t(), base.transpose(0, 1), base[:1].expand(3, 80, 130),
              base.view(2, 3, 80, 130), base[:, :1], base[:, :, :1], base.view(2, 3, 80, 130).permute(1, 0, 3, 2), base[:0]):
        got = ops.orthogonalise(x)
        assert got.shape == x.shape and got.dtype == dtype
        if x.numel():
            assert torch.equal(got, ops.orthogonalise(x.clone(memory_format=torch.contiguous_format)).view(got.shape)) or \
                float((got.double() - exact(x)).abs().max()) < 0.02      # (a transposed view runs the transposed iteration)
            check(got, x)


@DT
def test_a_list_of_matrices(dev, dtype):
    shapes = [(64, 294), (64, 576), (128, 64), (1, 9), (9, 1), (256, 700), (700, 256), (31, 31)] * 4      # more than one run of launches
    xs = [matrices(dev, s, dtype, i) for i, s in enumerate(shapes)]
    got = ops.orthogonalise(xs)
    for x, o in zip(xs, got):
        check(o, x)
    assert ops.orthogonalise([]) == []


def test_two_streams(dev):
    xs = [matrices(dev, (8, 200, 300), torch.float32, s) for s in (1, 2)]
    alone = [ops.orthogonalise(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = ops.orthogonalise(xs[i])
    torch.cuda.synchronize()
    assert torch.equal(alone[0], got[0]) and torch.equal(alone[1], got[1])


# ---- the step ---------------------------------------------------------------------------------------------------------------------------
def step_exact(w, g, m, lr, mu, nesterov, wd, gs=1.0, scale=None, steps=5):
    g = g.double() * gs
    m = mu * m.double() + g
    u = g + mu * m if nesterov else m
    f = max(1.0, w.shape[0] / w.shape[1]) ** 0.5 if scale is None else scale
    return (1 - lr * wd) * w.double() - lr * f * exact(u, steps), m, u, f


@DT
@pytest.mark.parametrize('nesterov', [True, False])
def test_muon_step(dev, dtype, nesterov):
    shapes = [(64, 294), (128, 64), (33, 65), (300, 200), (1, 40), (40, 1), (256, 1152)]
    ws = [matrices(dev, s, dtype, i) * 0.1 for i, s in enumerate(shapes)]
    ms = [matrices(dev, s, torch.float32, 50 + i) for i, s in enumerate(shapes)]
    for it in range(3):
        gs = [matrices(dev, s, dtype, 100 * it + i) for i, s in enumerate(shapes)]
        want = [step_exact(w, g, m, 0.05, 0.9, nesterov, 0.1, 0.5) for w, g, m in zip(ws, gs, ms)]
        ops.muon_step(ws, gs, ms, 0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1, grad_scale=0.5)
        for w, m, (w1, m1, u, f) in zip(ws, ms, want):
            assert float((m.double() - m1).abs().max()) <= 3 * 2.0 ** -24 * float(m1.abs().max() + 5)
            model = (noisy(u.float(), phases_of(dtype, 5)) - exact(u.float())).square().sum().sqrt()
            # u is rounded to fp32 (a step of it is within the model's noise), the sum once to the weight's type
            allowed = 0.05 * f * (12 * model + 2.0 ** -20 * exact(u).square().sum().sqrt()) + 1.1 * HALF[dtype] * w1.square().sum().sqrt()
            assert float((w.double() - w1).square().sum().sqrt()) <= float(allowed)


def test_muon_step_on_convolution_weights(dev):
    """Contiguous and channels-last weights (with gradient and momentum laid out alike) take the same step."""
    w = matrices(dev, (48, 20, 3, 3), torch.float32, 1)
    g, m = matrices(dev, (48, 20, 3, 3), torch.float32, 2), torch.zeros(48, 20, 3, 3, device=dev)
    a = [t.clone() for t in (w, g, m)]
    b = [t.clone(memory_format=torch.channels_last) for t in (w, g, m)]
    ops.muon_step([a[0]], [a[1]], [a[2]], 0.1)
    ops.muon_step([b[0]], [b[1]], [b[2]], 0.1)
    want = step_exact(w.flatten(1), g.flatten(1), m.flatten(1), 0.1, 0.95, True, 0.0)[0].view(w.shape)
    for got in (a, b):
        assert float((got[0].double() - want).abs().max()) < 0.1 * 2e-5
        assert float((got[2] - g).abs().max()) <= 2.0 ** -23 * float(g.abs().max())
    assert b[0].is_contiguous(memory_format=torch.channels_last)


def test_muon_step_on_pointwise_weights(dev):
    """A 1 x 1 convolution's gradient may carry other strides in its single-entry dimensions."""
    w, g, m = (matrices(dev, (24, 40, 1, 1), torch.float32, k) for k in range(3))
    a = [t.clone() for t in (w, g, m)]
    b = [w.clone(), g.clone().as_strided(g.shape, (40, 1, 40, 40)), m.clone()]
    ops.muon_step([a[0]], [a[1]], [a[2]], 0.1)
    ops.muon_step([b[0]], [b[1]], [b[2]], 0.1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


def test_learning_rate_that_changes_in_place(dev):
    w, g = matrices(dev, (20, 30), torch.float32, 1), matrices(dev, (20, 30), torch.float32, 2)
    lr, got, want = torch.tensor(0.1), w.clone(), w.clone()
    plan = ops.MuonUpdate([got], [g], [torch.zeros_like(w)])
    m = torch.zeros_like(w)
    for value in (0.1, 0.025):
        lr.fill_(value)
        plan.step(lr)
        ops.muon_step([want], [g], [m], float(lr))
        assert torch.equal(got, want)


def test_muon_step_leaves_the_rest_alone(dev):
    """Rows of a wider storage: what lies between them stays."""
    store = matrices(dev, (70, 200), torch.float32, 1)
    keep = store.clone()
    w = store[3:60, 10:150]
    g = matrices(dev, (57, 300), torch.float32, 2)[:, 5:145]
    m = torch.zeros(57, 140, device=dev)
    want = step_exact(w.clone(), g, m, 0.1, 0.95, True, 0.0)[0]
    ops.muon_step([w], [g], [m], 0.1)
    assert float((w.double() - want).abs().max()) < 1e-5
    store[3:60, 10:150] = keep[3:60, 10:150]
    assert torch.equal(store, keep)


def test_captured_steps(dev):
    """A captured step replays on the buffers' current contents, with eager work between the replays; two graphs do not share a workspace."""
    shapes = [(64, 200), (100, 80)]

    def state(seed):
        return [[matrices(dev, s, torch.float32, seed + 10 * k + i) for i, s in enumerate(shapes)] for k in range(3)]
    cap = [state(1), state(2)]
    ref = [state(1), state(2)]
    ops.muon_step(*state(3), 0.1)
    torch.cuda.synchronize()
    graphs = []
    for s in cap:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.muon_step(*s, 0.1, weight_decay=0.1)
        graphs.append(g)
    for k in range(3):
        for i in (0, 1):
            for a, b in zip(cap[i][1], ref[i][1]):
                new = matrices(dev, a.shape, torch.float32, 77 + k)
                a.copy_(new)
                b.copy_(new)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            ops.muon_step(*ref[i], 0.1, weight_decay=0.1)
            for a, b in zip(cap[i][0] + cap[i][2], ref[i][0] + ref[i][2]):
                assert torch.equal(a, b), (k, i)


def test_refusals(dev):
    x = torch.randn(4, 5, device=dev)
    for bad in (torch.randn(4, device=dev), torch.empty(0, 3, device=dev), torch.ones(3, 3, dtype=torch.int32, device=dev), x.double()):
        with pytest.raises(L.WgsError):
            ops.orthogonalise(bad)
    with pytest.raises(L.WgsError, match='no gradient'):
        ops.orthogonalise(x.clone().requires_grad_(True))
    with torch.no_grad():
        ops.orthogonalise(x.clone().requires_grad_(True))
    with pytest.raises(L.WgsError, match='steps'):
        ops.orthogonalise(x, steps=17)
    with pytest.raises(L.WgsError, match='bounded'):
        ops.orthogonalise(x, coefficients=(50.0, 3.0, 1.0))
    with pytest.raises(L.WgsError, match='share device and type'):
        ops.orthogonalise([x, x.half()])
    m = torch.zeros(4, 5, device=dev)
    with pytest.raises(L.WgsError, match='twice'):
        ops.muon_step([x, x], [x.clone(), x.clone()], [m, m.clone()], 0.1)
    with pytest.raises(L.WgsError, match='overlaps'):
        ops.muon_step([x], [x], [m], 0.1)                                   # a gradient that is the weight
    with pytest.raises(L.WgsError, match='overlaps'):
        ops.muon_step([x], [m], [m], 0.1)
    big = torch.randn(12, 5, device=dev)
    with pytest.raises(L.WgsError, match='overlaps'):
        ops.muon_step([big[:8], big[6:10]], [torch.randn(8, 5, device=dev), x], [torch.zeros(8, 5, device=dev), m], 0.1)
    w = torch.nn.Parameter(x.clone())
    plan = ops.MuonUpdate([w], [x], [m])
    plan.step(0.1)
    w.data = w.data.clone()
    with pytest.raises(L.WgsError, match='other memory'):
        plan.step(0.1)
    g = x.clone()
    with pytest.raises(L.WgsError, match='momentum must be'):
        ops.muon_step([x], [g], [m], 0.1, momentum=1.0)
    with pytest.raises(L.WgsError, match='a momentum must be'):
        ops.muon_step([x], [x], [m.half()], 0.1)
    with pytest.raises(L.WgsError, match='elements of a row'):
        ops.muon_step([x.t()], [x.t()], [torch.zeros(5, 4, device=dev)], 0.1)
