"""Label log-probabilities, entropy, top alternatives and their gradient against the formulas in 64 bits."""
import math

import pytest
import torch

from warpedganspace_amd import _lib as L
from warpedganspace_amd import ops

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24                 # half a step of fp32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # a step below the normal range


def reference(logits, labels, top, ignore=-100):
    x = logits.detach().double().cpu()
    lab = labels.cpu()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    ent = torch.special.entr(p).sum(-1)
    ok = (lab != ignore) & (lab >= 0) & (lab < x.shape[-1])
    at = torch.where(ok, lab, torch.zeros_like(lab))
    lp = torch.where(ok, logp.gather(-1, at.unsqueeze(-1)).squeeze(-1), torch.zeros_like(ent))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
    return lp, ent, logp.gather(-1, order), order, logp, p


def delta(V):
    """Bound of the relative error of s = sum exp(l - m), which is the absolute one of log s.  A term's: the rounding of (l - m) log2 e
    times ln 2, |l - m| 2^-23 (weighted by its share: below 32 for every term that counts), and a step of exp2; a lane adds V / 64 terms at
    most (one wave a row up to 2048 scores; else V / 256), then a tree of at most 6 + 3 + 6 joins of two products each."""
    chain = V / 64 if V <= 2048 else V / 256
    return EPS * (chain + 64 + 4 + 3 * 15)


def close(got, want, bound, what):
    got = got.detach().double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    err = (got - want).abs()
    bad = ~(same | (err <= bound))
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float((err / bound)[bad].max()))


def check(logits, labels, top, ignore=-100, g=None, h=None, q=None):
    V = logits.shape[-1]
    lp, ent, tl, ti, logp, p = reference(logits, labels, top, ignore)
    r = ops.label_logprobs(logits, labels, top=top, ignore_index=ignore)
    d = delta(V)
    close(r.logp, lp, d + 4 * EPS * lp.abs(), 'logp')
    # H = log s - u / s, |u / s| = E|l - m| <= H + log V: u has the relative error of s and a rounding of each product
    close(r.entropy, ent, (2 * d + 8 * EPS) * (1 + ent + math.log(V)), 'entropy')
    close(r.top_logp, tl, d + 4 * EPS * tl.abs(), 'top_logp')
    assert torch.equal(r.top_index.cpu(), ti)
    if g is None:
        return r
    grad, = torch.autograd.grad([r.logp, r.entropy, r.top_logp], [logits], [g, h, q])
    g, h, q = (t.double().cpu().unsqueeze(-1) for t in (g, h, q))
    lab = labels.cpu()
    gl = torch.where((lab == ignore).unsqueeze(-1), torch.zeros_like(g), g)
    total = gl + q.squeeze(-1).sum(-1, keepdim=True)
    lf = logp.clamp(min=-1e5)
    E = ent.unsqueeze(-1)
    want = -p * (total + h * (lf + E))
    add = torch.zeros_like(want)
    add.scatter_add_(-1, torch.where((lab == ignore), torch.zeros_like(lab), lab).unsqueeze(-1), gl)
    add.scatter_add_(-1, ti, q.squeeze(-1))
    want = want + add
    # p has the relative error d + |log p| steps; the bracket that of its terms; then the sum with the row's own terms and the rounding
    mag = total.abs() + h.abs() * (lf.abs() + E + math.log(V)) + q.squeeze(-1).abs().sum(-1, keepdim=True)
    bound = p * mag * (2 * d + 12 * EPS + 4 * EPS * lf.abs().clamp(max=200)) + 4 * EPS * (add.abs() + gl.abs() * (add != 0))
    bound = bound + HALF[logits.dtype] * (want.abs() + bound) + TINY[logits.dtype] + 1e-37
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    close(grad, want, bound, 'grad')
    return r


def make(dev, rows, V, dtype, seed, pad=0, scale=3.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, V + pad, generator=gen, device=dev) * scale).to(dtype)[:, :V]
    labels = torch.randint(0, V, (rows,), generator=gen, device=dev)
    return x.requires_grad_(True), labels, gen


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows,V,top,pad', [
    (1, 1, 1, 0), (3, 2, 2, 0), (32, 128, 5, 0), (33, 200, 64, 3), (5, 63, 63, 1), (7, 2047, 20, 0), (6, 2048, 1, 5), (5, 2049, 20, 0),
    (2, 8191, 64, 0), (1, 40007, 20, 0), (9, 32000, 0, 0), (600, 5003, 3, 2), (4, 131072, 20, 0), (1, 262139, 64, 0)])
def test_values_and_gradient(dev, dtype, rows, V, top, pad):
    x, labels, gen = make(dev, rows, V, dtype, rows * 7 + V, pad)
    labels[::4] = -100
    g = torch.randn(rows, generator=gen, device=dev)
    h = torch.randn(rows, generator=gen, device=dev)
    q = torch.randn(rows, top, generator=gen, device=dev)
    check(x, labels, top, g=g, h=h, q=q)


@pytest.mark.parametrize('V', [4097, 4098, 8193, 8195, 16385, 16390, 24577])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
def test_last_classes_of_rows_at_every_alignment(dev, dtype, V):
    """A row whose vectors end with a workgroup's part and that has scores left behind them: their own terms belong to the last workgroup."""
    x, labels, gen = make(dev, 24, V, dtype, V)
    labels[:] = V - 1 - torch.arange(24, device=dev) % 3
    with torch.no_grad():
        x[:, -3:] += 15.0                       # alternatives too
    g, h, q = (torch.randn(s, generator=gen, device=dev) for s in ((24,), (24,), (24, 4)))
    check(x, labels, 4, g=g, h=h, q=q)
    # the gradient at another place of a 16-byte block than the scores: one score at a time
    r = ops.label_logprobs(x, labels, top=4)
    want, = torch.autograd.grad([r.logp, r.entropy, r.top_logp], [x], [g, h, q])
    r = ops.label_logprobs(x, labels, top=4)
    stat = r.logp.grad_fn.saved_tensors[2]
    out = torch.full((24, V + 3), 7.0, dtype=dtype, device=dev)
    L.check(ops._logprobs()[2](x.data_ptr(), ops._DTYPES[dtype], 24, V, V, labels.data_ptr(), -100, stat.data_ptr(), r.entropy.data_ptr(), 4,
                               r.top_index.data_ptr(), g.data_ptr(), h.data_ptr(), q.data_ptr(), out.data_ptr() + out.element_size(), V + 3, L.stream_id()),
            'wgs_label_logprobs_bwd')
    assert torch.equal(out[:, 1:V + 1], want) and (out[:, V + 1:] == 7).all() and (out[:, :1] == 7).all()


@pytest.mark.parametrize('V', [40, 1000, 4099, 70001])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_masked_scores(dev, dtype, V):
    """-inf and the type's lowest value in masked places, rows of one allowed class, rows with fewer allowed classes than alternatives."""
    x, labels, gen = make(dev, 8, V, dtype, V)
    x = x.detach()
    x[0, 1:] = -math.inf
    x[1, :-1] = -math.inf
    x[2, 5:] = torch.finfo(dtype).min
    x[3, :] = torch.finfo(dtype).min
    x[4, V // 2:] = -math.inf
    x[5, ::2] = -math.inf
    x[6] = 7.0
    labels[0], labels[1] = 0, 0
    x.requires_grad_(True)
    one = torch.ones(8, device=dev)
    r = check(x, labels, 20, g=one, h=0.5 * one, q=torch.zeros(8, 20, device=dev))
    assert r.logp[0] == 0 and r.entropy[0] == 0 and r.logp[1] == -math.inf


@pytest.mark.parametrize('V', [33, 5000, 66000])
def test_empty_and_broken_rows(dev, V):
    x, labels, gen = make(dev, 5, V, torch.float32, V)
    x = x.detach()
    x[0] = -math.inf
    x[1, V // 3] = math.nan
    x[2, V - 1] = math.inf
    labels[3] = V
    labels[4] = -1
    x.requires_grad_(True)
    r = ops.label_logprobs(x, labels, top=3)
    assert r.logp[0] == -math.inf and r.entropy[0] == 0 and r.top_index[0].tolist() == [0, 1, 2] and (r.top_logp[0] == -math.inf).all()
    for b in (1, 2):
        assert r.logp[b].isnan() and r.entropy[b].isnan() and r.top_logp[b].isnan().all() and r.top_index[b].tolist() == [-1] * 3
    assert r.logp[3].isnan() and r.logp[4].isnan() and not r.entropy[3:].isnan().any()
    grad, = torch.autograd.grad([r.logp.sum() + r.entropy.sum()], [x])
    assert (grad[0] == 0).all() and grad[1].isnan().all() and grad[2].isnan().all() and grad[3].isnan().all() and grad[4].isnan().all()


@pytest.mark.parametrize('V', [64, 1500, 9000, 131072])
@pytest.mark.parametrize('kind', ['all equal', 'few values', 'ascending', 'descending', 'zeros of both signs'])
def test_equal_scores_come_in_the_order_of_their_indices(dev, V, kind):
    gen = torch.Generator(device=dev).manual_seed(V)
    if kind == 'all equal':
        x = torch.full((2, V), -1.5, device=dev)
    elif kind == 'few values':
        x = torch.randint(0, 4, (2, V), generator=gen, device=dev).float()
    elif kind == 'zeros of both signs':
        x = torch.where(torch.rand(2, V, generator=gen, device=dev) < 0.5, 0.0, -0.0)
    else:
        x = torch.arange(V, device=dev).float().expand(2, V).contiguous() / V
        x = x.flip(1).contiguous() if kind == 'descending' else x
    check(x, torch.zeros(2, dtype=torch.int64, device=dev), 40)


def test_shapes_and_strides(dev):
    x = torch.randn(3, 4, 50, device=dev)
    labels = torch.randint(0, 50, (3, 4), device=dev)
    for y, lab in ((x, labels), (x.transpose(0, 1), labels.t()), (x[:, :, ::2], labels % 25), (x[:, 1:3, 7:], labels[:, 1:3] % 43),
                   (x[0, 0], labels[0, 0]), (x[:1].expand(5, 4, 50), labels[:1].expand(5, 4)), (x.permute(2, 0, 1)[:, :, :], None)):
        if lab is None:
            lab = torch.randint(0, y.shape[-1], y.shape[:-1], device=dev)
        y = y.detach().requires_grad_(True)
        assert y.is_leaf
        z = torch.ones(lab.shape, device=dev)
        check(y, lab, 2, g=z, h=0.3 * z, q=torch.zeros(*lab.shape, 2, device=dev))
    empty = ops.label_logprobs(torch.empty(0, 50, device=dev), torch.empty(0, dtype=torch.int64, device=dev), top=2)
    assert empty.logp.shape == (0,) and empty.top_index.shape == (0, 2)


def test_odd_addresses(dev):
    """Rows that begin inside a 16-byte block, in storage and out of it; a row's neighbours are not touched by the gradient."""
    for dtype in (torch.float32, torch.bfloat16):
        for first in (1, 3, 5):
            store = torch.randn(first + 6 * 3001, device=dev).to(dtype)
            x = store[first:].view(6, 3001)[:, :2999].requires_grad_(True)
            labels = torch.randint(0, 2999, (6,), device=dev)
            z = torch.ones(6, device=dev)
            check(x, labels, 4, g=z, h=z, q=torch.ones(6, 4, device=dev))


def test_far_scores_keep_their_differences(dev):
    x = (torch.randn(4, 3000, device=dev) + 8192).to(torch.float32).requires_grad_(True)
    labels = torch.randint(0, 3000, (4,), device=dev)
    z = torch.ones(4, device=dev)
    check(x, labels, 5, g=z, h=z, q=torch.zeros(4, 5, device=dev))


def test_gradient_against_differences(dev):
    """Central differences of a weighted sum of all outputs, f, along one direction: f''' h^2 / 6 with |f'''| <= 10 |w| |dir|_inf^3 of the
    softmax's moments, and the rounding of both values over 2 h."""
    V, h = 300, 2.0 ** -6
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(1, V, generator=gen, device=dev)
    x[0, :3] += torch.tensor([6.0, 5.0, 4.0], device=dev)      # the alternatives stay the same within +-h
    labels = torch.tensor([17], device=dev)
    direction = torch.rand(1, V, generator=gen, device=dev) * 2 - 1

    def f(y):
        r = ops.label_logprobs(y, labels, top=3)
        return 1.5 * r.logp.sum() - 0.5 * r.entropy.sum() + (r.top_logp * torch.tensor([[1.0, -2.0, 0.5]], device=dev)).sum()
    y = x.clone().requires_grad_(True)
    grad, = torch.autograd.grad(f(y), y)
    with torch.no_grad():
        diff = (f(x + h * direction).double() - f(x - h * direction).double()) / (2 * h)
    want = (grad.double() * direction.double()).sum()
    assert abs(float(diff - want)) <= 10 * 6 * h * h / 6 + 16 * delta(V) * 6 / (2 * h), (float(diff), float(want))


def test_two_streams_and_another_order(dev):
    """Two calls at once on streams of their own give what they give alone, bit for bit."""
    xs = [make(dev, 16, 50000, torch.bfloat16, s)[:2] for s in (1, 2)]
    alone = [ops.label_logprobs(x, l, top=20) for x, l in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = ops.label_logprobs(*xs[i], top=20)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


def test_captured_and_replayed(dev):
    x, labels, gen = make(dev, 8, 40000, torch.float16, 5)
    x = x.detach().clone().requires_grad_(True)
    g = torch.randn(8, generator=gen, device=dev)

    def call():
        r = ops.label_logprobs(x, labels, top=6)
        return (r.logp, r.entropy, r.top_logp, r.top_index) + torch.autograd.grad([r.logp, r.entropy], [x], [g, g])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(8, 40000, generator=gen, device=dev) * (k + 1))
            labels.copy_(torch.randint(0, 40000, (8,), generator=gen, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, call()):
            assert torch.equal(a, b), k


def test_long_rows_past_32_bits(dev):
    """Scores of the last rows lie more than 2^31 elements behind the first one."""
    rows, V = 3, 70000
    store = torch.zeros((1 << 31) + 400000, dtype=torch.bfloat16, device=dev)
    stride = ((1 << 31) + 8 * 1024) // 2
    x = store.as_strided((rows, V), (stride, 1))
    src = (torch.randn(rows, V, device=dev) * 3).to(torch.bfloat16)
    x.copy_(src)
    labels = torch.randint(0, V, (rows,), device=dev)
    far, near = ops.label_logprobs(x, labels, top=5), ops.label_logprobs(src, labels, top=5)
    for a, b in zip(far, near):
        assert torch.equal(a, b)
